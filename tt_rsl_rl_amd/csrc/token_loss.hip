// Token log-probabilities and the clipped policy loss with a KL term, forward and gradient (ppo_token_log_probs,
// ppo_token_ppo_loss): the categorical counterpart of loss.hip's Gaussian head.
//
// With c = log2(e) / temperature, m = max_j x_j and t_j = c (x_j - m) (the difference first: where every logit is the type's
// lowest value c m alone would overflow):
//   S = sum_j 2^t_j,  E = sum_j 2^t_j t_j,  lp = ln2 (t_token - log2 S),  H = ln2 (log2 S - E / S),
//   p_j = 2^w_j with w_j = t_j - log2 S,  d_logits_j = p_j (a + b w_j) + [j = token] g k,
//   k = 1 / (N temperature),  a = k (entropy_coef H - g),  b = k entropy_coef ln2.
// A logit of -inf has 2^t = 0 exactly; its t and w are raised to kFloor, where 2^kFloor is 0 too, so that 0 t stays 0.
// Bound by memory: the logits once in, their gradient once out.
#include "elem.hpp"

namespace ppo {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1000.0f;
constexpr int kThreads = 256;
constexpr int kTerms = 5;  // per row: s, k, H, clipped, old_logp - lp

struct LossKernelArgs {
  ppo_token_loss_args a;
  float* inv_n;   // 1 / N (0: no row counts)
  float* n;
  float* terms;   // [kTerms][rows]
  float c, inv_temp, clip_lo, clip_hi, kl_coef, entropy_coef;
};

__device__ __forceinline__ bool counts(const ppo_token_loss_args& a, int64_t r, int64_t& tok) {
  tok = -1;
  if (a.mask != nullptr && a.mask[r] == 0) return false;
  tok = token_at(a.tokens, a.token_type, r, a.vocab);
  return tok >= 0;
}

template <class R>
__device__ __forceinline__ R wave_sum(R x) {
  for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_xor(x, d, kWave);
  return x;
}

__global__ __launch_bounds__(1024) void token_count_kernel(const LossKernelArgs q) {
  __shared__ int32_t part[1024 / kWave];
  int32_t n = 0;
  int64_t tok;
  for (int64_t r = threadIdx.x; r < q.a.rows; r += 1024) n += counts(q.a, r, tok) ? 1 : 0;
  n = wave_sum(n);
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int64_t all = 0;
    for (int w = 0; w < 1024 / kWave; ++w) all += part[w];
    const double d = q.a.denom > 0.0 ? q.a.denom : static_cast<double>(all);
    *q.n = static_cast<float>(d);
    *q.inv_n = all > 0 ? static_cast<float>(1.0 / d) : 0.0f;
  }
}

// Sum (or maximum) over the block, in every thread.
template <class F>
__device__ __forceinline__ float block_reduce(float x, float* scratch, F&& f) {
  for (int d = kWave / 2; d > 0; d >>= 1) x = f(x, __shfl_xor(x, d, kWave));
  if (threadIdx.x % kWave == 0) scratch[threadIdx.x / kWave] = x;
  __syncthreads();
  x = scratch[0];
  for (int w = 1; w < kThreads / kWave; ++w) x = f(x, scratch[w]);
  __syncthreads();
  return x;
}

// The row's scalars once S and E are known; writes logp, entropy and the loss terms. Returns g (the derivative by lp).
struct RowScalars {
  float log2_s, h, g;
};

__device__ __forceinline__ RowScalars row_scalars(const LossKernelArgs& q, int64_t r, float t_tok, float s, float e, bool loss,
                                                  bool write) {
  RowScalars o;
  o.log2_s = log2f(s);
  const float lp = kLn2 * (t_tok - o.log2_s);
  o.h = kLn2 * (o.log2_s - e / s);
  o.g = 0.0f;
  if (write && q.a.logp != nullptr) q.a.logp[r] = lp;
  if (write && q.a.entropy != nullptr) q.a.entropy[r] = o.h;
  if (!loss) return o;
  const float old = q.a.old_logp[r], adv = q.a.advantages[r];
  const float ratio = expf(lp - old);
  const float clipped = fminf(fmaxf(ratio, q.clip_lo), q.clip_hi);
  const float first = -adv * ratio, second = -adv * clipped;
  float kl = 0.0f;
  o.g = first >= second ? first : first < second ? 0.0f : first + second;  // (NaN goes on)
  if (q.a.ref_logp != nullptr) {
    const float d = q.a.ref_logp[r] - lp, x = expf(d);
    kl = x - d - 1.0f;
    o.g += q.kl_coef * (1.0f - x);
  }
  if (write) {
    const int64_t n = q.a.rows;
    q.terms[r] = first != first || second != second ? first + second : fmaxf(first, second);
    q.terms[n + r] = kl;
    q.terms[2 * n + r] = o.h;
    q.terms[3 * n + r] = ratio != clipped ? 1.0f : 0.0f;
    q.terms[4 * n + r] = old - lp;
  }
  return o;
}

__device__ __forceinline__ void row_zeros(const LossKernelArgs& q, int64_t r, bool loss) {
  if (q.a.logp != nullptr) q.a.logp[r] = 0.0f;
  if (q.a.entropy != nullptr) q.a.entropy[r] = 0.0f;
  if (loss)
    for (int i = 0; i < kTerms; ++i) q.terms[i * q.a.rows + r] = 0.0f;
}

// One block per row, the row read three times: its maximum, its sums, its gradient.
template <class T, bool LOSS>
__global__ __launch_bounds__(kThreads) void token_row_kernel(const LossKernelArgs q) {
  __shared__ float scratch[kThreads / kWave];
  const ppo_token_loss_args& a = q.a;
  const int64_t r = blockIdx.x;
  const T* x = static_cast<const T*>(a.logits) + r * a.ld_logits;
  T* dx = LOSS && a.d_logits != nullptr ? static_cast<T*>(a.d_logits) + r * a.ld_d_logits : nullptr;
  int64_t tok;
  bool live = counts(a, r, tok);
  float m = -INFINITY;
  if (live) {
    for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) m = fmaxf(m, static_cast<float>(x[j]));
    m = block_reduce(m, scratch, [](float u, float v) { return fmaxf(u, v); });
    // -inf throughout (a NaN among them still goes on): no distribution
    if (m == -INFINITY) {
      float nan = 0.0f;
      for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) nan += x[j] != x[j] ? 1.0f : 0.0f;
      live = block_reduce(nan, scratch, [](float u, float v) { return u + v; }) > 0.0f;
    }
  }
  if (!live) {
    if (threadIdx.x == 0) row_zeros(q, r, LOSS);
    if (dx != nullptr)
      for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) dx[j] = static_cast<T>(0.0f);
    return;
  }
  float s = 0.0f, e = 0.0f;
  for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) {
    const float t = (static_cast<float>(x[j]) - m) * q.c, p = exp2f(t);
    s += p;
    e = fmaf(p, fmaxf(t, kFloor), e);
  }
  s = block_reduce(s, scratch, [](float u, float v) { return u + v; });
  e = block_reduce(e, scratch, [](float u, float v) { return u + v; });
  const float t_tok = (static_cast<float>(x[tok]) - m) * q.c;
  const RowScalars o = row_scalars(q, r, t_tok, s, e, LOSS, threadIdx.x == 0);
  if (dx == nullptr) return;
  const float k = *q.inv_n * q.inv_temp;
  const float ca = k * (q.entropy_coef * o.h - o.g), cb = k * q.entropy_coef * kLn2, ct = k * o.g;
  __syncthreads();  // x[tok] has been read by every thread: d_logits may be the logits
  for (int64_t j = threadIdx.x; j < a.vocab; j += kThreads) {
    const float w = fmaxf((static_cast<float>(x[j]) - m) * q.c - o.log2_s, kFloor);
    float d = exp2f(w) * fmaf(cb, w, ca);
    if (j == tok) d += ct;
    dx[j] = static_cast<T>(d);
  }
}

// The means over rows, fp64 sums in a fixed order.
__global__ __launch_bounds__(1024) void token_stats_kernel(const LossKernelArgs q) {
  __shared__ double part[kTerms][1024 / kWave];
  double sum[kTerms] = {};
  for (int64_t r = threadIdx.x; r < q.a.rows; r += 1024)
#pragma unroll
    for (int i = 0; i < kTerms; ++i) sum[i] += static_cast<double>(q.terms[i * q.a.rows + r]);
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    const double x = wave_sum(sum[i]);
    if (threadIdx.x % kWave == 0) part[i][threadIdx.x / kWave] = x;
  }
  __syncthreads();
  if (threadIdx.x != 0) return;
  const double inv = *q.inv_n > 0.0f ? 1.0 / static_cast<double>(*q.n) : 0.0;
  double mean[kTerms];
  for (int i = 0; i < kTerms; ++i) {
    double x = 0.0;
    for (int w = 0; w < 1024 / kWave; ++w) x += part[i][w];
    mean[i] = x * inv;
  }
  q.a.stats[0] = static_cast<float>(mean[0] + q.a.kl_coef * mean[1] - q.a.entropy_coef * mean[2]);
  for (int i = 0; i < kTerms; ++i) q.a.stats[1 + i] = static_cast<float>(mean[i]);
  q.a.stats[6] = *q.n;
  q.a.stats[7] = 0.0f;
}

size_t workspace_for(int64_t rows) {
  return (64 + static_cast<size_t>(kTerms) * static_cast<size_t>(rows)) * sizeof(float);
}

int run(const char* who, const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream,
        bool loss) {
  PPO_REQUIRE(args != nullptr, "%s: null arguments", who);
  const ppo_token_loss_args& a = *args;
  PPO_REQUIRE(a.rows >= 0 && a.rows < INT32_MAX && a.vocab >= 1 && a.vocab < INT32_MAX, "%s: rows=%lld vocab=%lld", who,
              (long long)a.rows, (long long)a.vocab);
  PPO_REQUIRE(type_ok(a.type), "%s: type=%d", who, a.type);
  PPO_REQUIRE(a.token_type == PPO_TOKENS_I64 || a.token_type == PPO_TOKENS_I32, "%s: token_type=%d", who, a.token_type);
  PPO_REQUIRE(a.temperature > 0.0 && a.temperature < 1e30, "%s: temperature=%g", who, a.temperature);
  PPO_REQUIRE(a.ld_logits >= a.vocab && (!loss || a.d_logits == nullptr || a.ld_d_logits >= a.vocab),
              "%s: leading dimensions below vocab=%lld", who, (long long)a.vocab);
  PPO_REQUIRE(a.rows == 0 || (a.logits != nullptr && a.tokens != nullptr), "%s: null pointer", who);
  const size_t align = type_size(a.type);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a.logits) % align == 0 && reinterpret_cast<uintptr_t>(a.d_logits) % align == 0 &&
                  reinterpret_cast<uintptr_t>(a.tokens) % (a.token_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  if (loss) {
    PPO_REQUIRE(a.stats != nullptr && (a.rows == 0 || (a.old_logp != nullptr && a.advantages != nullptr)),
                "%s: null pointer", who);
    PPO_REQUIRE(a.clip_low >= 0.0 && a.clip_high >= 0.0, "%s: clip range %g, %g", who, a.clip_low, a.clip_high);
    PPO_REQUIRE(a.denom >= 0.0 && a.denom < 1e30, "%s: denom=%g", who, a.denom);
    const size_t need = workspace_for(a.rows);
    PPO_REQUIRE(workspace != nullptr && workspace_bytes >= need, "%s: workspace too small (%zu < %zu)", who,
                workspace_bytes, need);
    PPO_REQUIRE(a.d_logits != a.logits || a.ld_d_logits == a.ld_logits, "%s: in place needs the same rows", who);
  } else if (a.rows == 0 || (a.logp == nullptr && a.entropy == nullptr)) {
    return PPO_OK;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  LossKernelArgs q{};
  q.a = a;
  q.inv_n = static_cast<float*>(workspace);
  q.n = q.inv_n + 1;
  q.terms = q.inv_n + 64;
  q.inv_temp = static_cast<float>(1.0 / a.temperature);
  q.c = static_cast<float>(1.4426950408889634 / a.temperature);
  q.clip_lo = static_cast<float>(1.0 - a.clip_low);
  q.clip_hi = static_cast<float>(1.0 + a.clip_high);
  q.kl_coef = static_cast<float>(a.kl_coef);
  q.entropy_coef = static_cast<float>(a.entropy_coef);
  if (loss) {
    hipLaunchKernelGGL(token_count_kernel, dim3(1), dim3(1024), 0, st, q);
    if (int rc = check_launch("token_count_kernel")) return rc;
  }
  if (a.rows > 0) {
    int rc = PPO_OK;
    with_type(a.type, [&](auto t) {
      using T = decltype(t);
      const dim3 grid(static_cast<uint32_t>(a.rows));
      if (loss) hipLaunchKernelGGL((token_row_kernel<T, true>), grid, dim3(kThreads), 0, st, q);
      else hipLaunchKernelGGL((token_row_kernel<T, false>), grid, dim3(kThreads), 0, st, q);
      rc = check_launch("token_row_kernel");
    });
    if (rc != PPO_OK) return rc;
  }
  if (!loss) return PPO_OK;
  hipLaunchKernelGGL(token_stats_kernel, dim3(1), dim3(1024), 0, st, q);
  return check_launch("token_stats_kernel");
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_token_loss_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows >= INT32_MAX || vocab < 1 || vocab >= INT32_MAX) return 0;
  return workspace_for(rows);
}

extern "C" int ppo_token_log_probs(const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes,
                                   ppo_stream_t stream) {
  return run("ppo_token_log_probs", args, workspace, workspace_bytes, stream, false);
}

extern "C" int ppo_token_ppo_loss(const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes,
                                  ppo_stream_t stream) {
  return run("ppo_token_ppo_loss", args, workspace, workspace_bytes, stream, true);
}
