// AdamW over a list of tensors (ppo_adamw_step): clip by the global norm, then the update, states in 32 or in 8 bits.
//
//   1. sums of squares of the gradients, fp64, one partial per block;
//   2. one block adds the partials in order: total and the clip coefficient (both left out without a clip);
//   3. the update, chunks of a tensor per block.
// The tensors' addresses travel as kernel arguments, kMaxTensors to a launch, so nothing about a call is kept on the device.
// The element update is optim.hip's, torch's fp32 operation order with contraction disabled.
//
// States in 8 bits: 256 consecutive elements share an fp32 scale per state; m = +-scale (|q| / 127)^2, v = scale (q / 255)^4.
// The powers place codes densely near zero, as the magnitudes lie: the smallest m but zero is 6e-5 of the block's largest, the
// smallest sqrt(v) 1.5e-5 of it.  A wave owns a block of elements, four per lane, so the new scale is one wave reduction.
// A step of beta2 = 0.999 lowers v by 0.1 % at most, and neighbouring codes of v lie 1.6 % or more apart: rounded to nearest, a v
// below its block's largest never falls (gradients of half a block a tenth of what they were: 5,000 steps later their v is 82
// times too large).  With `dither` a code is rounded up or down by chance, so that what it stands for is the value on average and
// the moments follow (1.005 times, by the same count).
//
// Bound by memory: 28 bytes per fp32 parameter with fp32 states, and the gradient once more for the norm.
// 60 M bf16 with masters: update 269 us, 6.2 TB/s, norm 25; 250 M with 8-bit states: update 705 us, 5.8 TB/s, norm 114; with
// dither the update is bound by its arithmetic (a step without a norm 804 us, 715 to nearest).
#include "elem.hpp"

#pragma clang fp contract(off)

namespace ppo {
namespace {

constexpr int kAdamwThreads = 256, kPer = 4;
constexpr int kChunk = kAdamwThreads * kPer;  // elements a block takes at a time
constexpr int kMaxTensors = 41, kMaxGrads = 160;
constexpr int kNormChunk = 8 * kChunk, kNormBlocks = 2048;  // elements a block's loads have in flight, blocks of one norm launch
static_assert(kChunk % PPO_ADAMW_BLOCK == 0 && PPO_ADAMW_BLOCK == kWave * kPer, "a wave owns a scale's block");

struct NormTable {
  const void* grad[kMaxGrads];
  int64_t count[kMaxGrads];
  int32_t first[kMaxGrads + 1];  // chunks before the tensor
  int32_t tensors;
};
static_assert(sizeof(NormTable) <= 3800, "kernel arguments");

struct Tensor {
  void* param;
  const void* grad;
  float* master;
  void* m;
  void* v;
  float* m_scale;
  float* v_scale;
  int64_t count;
  float neg_step, decay, bc2_sqrt, inv_bc2_sqrt;
  uint32_t key;  // of the dither
};

struct UpdateTable {
  Tensor t[kMaxTensors];
  int32_t first[kMaxTensors + 1];
  int32_t tensors;
};
static_assert(sizeof(UpdateTable) <= 3800, "kernel arguments");

struct Scalars {
  float w1, b2, c2, eps;
};

// The tensor of a chunk: the last one whose first chunk is not behind it.
template <int N>
__device__ __forceinline__ int tensor_of(const int32_t (&first)[N], int tensors, int chunk) {
  int lo = 0, hi = tensors;
  while (hi - lo > 1) {
    const int mid = (lo + hi) / 2;
    if (first[mid] <= chunk) lo = mid;
    else hi = mid;
  }
  return lo;
}

__device__ __forceinline__ double block_sum(double x, double* red) {
  for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_down(x, d, kWave);
  if (threadIdx.x % kWave == 0) red[threadIdx.x / kWave] = x;
  __syncthreads();
  double s = 0.0;
  for (int w = 0; w < kAdamwThreads / kWave; ++w) s += red[w];
  __syncthreads();
  return s;
}

// Four elements from p, those past n as zeros.
template <bool STREAM, class T>
__device__ __forceinline__ void load4(const T* p, int n, float (&x)[kPer]) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (n >= kPer) {
    const vec* q = reinterpret_cast<const vec*>(p);
    vec v;
    if constexpr (STREAM) v = __builtin_nontemporal_load(q);
    else v = *q;
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = static_cast<float>(v[i]);
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i) x[i] = i < n ? static_cast<float>(p[i]) : 0.0f;
  }
}

template <bool STREAM, class T>
__device__ __forceinline__ void store4(T* p, int n, const float (&x)[kPer]) {
  typedef T vec __attribute__((ext_vector_type(4), aligned(sizeof(T))));
  if (n >= kPer) {
    vec v;
#pragma unroll
    for (int i = 0; i < kPer; ++i) v[i] = static_cast<T>(x[i]);
    if constexpr (STREAM) __builtin_nontemporal_store(v, reinterpret_cast<vec*>(p));
    else *reinterpret_cast<vec*>(p) = v;
  } else {
#pragma unroll
    for (int i = 0; i < kPer; ++i)
      if (i < n) p[i] = static_cast<T>(x[i]);
  }
}

template <class G>
__global__ __launch_bounds__(kAdamwThreads) void adamw_norm_kernel(const NormTable t, int chunks, double* __restrict__ partial) {
  constexpr int V = kVec<G>, K = kNormChunk / (kAdamwThreads * V);
  __shared__ double red[kAdamwThreads / kWave];
  double sum[4] = {};
  for (int c = blockIdx.x; c < chunks; c += gridDim.x) {
    const int k = tensor_of(t.first, t.tensors, c);
    const G* g = static_cast<const G*>(t.grad[k]);
    const int64_t from = static_cast<int64_t>(c - t.first[k]) * kNormChunk;
    const int left = static_cast<int>(min<int64_t>(kNormChunk, t.count[k] - from));
    g += from;
    // (the pieces of a tensor's last chunk are in flight together too: with its elements one after another a thread waited for up
    // to 32 loads in a row, and 150 tensors of 60 M bf16 took 39 us, 25 now)
    RawPiece x[K];
#pragma unroll
    for (int i = 0; i < K; ++i) {
      const int at = (i * kAdamwThreads + static_cast<int>(threadIdx.x)) * V;
      x[i] = at + V <= left ? load_raw(g + at) : RawPiece{};
    }
    const int rest = left / V * V + static_cast<int>(threadIdx.x);  // the elements behind the last whole piece
    const double odd = rest < left ? static_cast<double>(static_cast<float>(g[rest])) : 0.0;
    sum[0] = fma(odd, odd, sum[0]);
#pragma unroll
    for (int i = 0; i < K; ++i)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const double d = element<G>(x[i], e);
        sum[e % 4] = fma(d, d, sum[e % 4]);
      }
  }
  const double all = block_sum((sum[0] + sum[1]) + (sum[2] + sum[3]), red);
  if (threadIdx.x == 0) partial[blockIdx.x] = all;
}

// coef[0] = the clip coefficient
__global__ __launch_bounds__(kAdamwThreads) void adamw_clip_kernel(const double* __restrict__ partial, int partials, float max_norm,
                                                                   float* __restrict__ coef, float* __restrict__ norm_out) {
  __shared__ double red[kAdamwThreads / kWave];
  double sum = 0.0;
  for (int i = threadIdx.x; i < partials; i += kAdamwThreads) sum += partial[i];
  sum = block_sum(sum, red);
  if (threadIdx.x != 0) return;
  const float total = static_cast<float>(sqrt(sum));
  float c = 1.0f;
  if (max_norm > 0.0f) {
    c = max_norm / (total + 1e-6f);
    c = c > 1.0f ? 1.0f : c;  // (NaN stays)
  }
  coef[0] = c;
  if (norm_out != nullptr) {
    norm_out[0] = total;
    norm_out[1] = c;
  }
}

__device__ __forceinline__ float wave_max(float x) {
  for (int d = kWave / 2; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, kWave));
  return x;
}

// A block's new scale: the largest of its values (none negative); NaN where one is not finite, so that the block does not
// come back as if it were.
__device__ __forceinline__ float block_scale(const float (&x)[kPer]) {
  float s = 0.0f;
  bool bad = false;
#pragma unroll
  for (int i = 0; i < kPer; ++i) {
    s = fmaxf(s, x[i]);
    bad |= !(x[i] < INFINITY);
  }
  s = wave_max(s);
  return __ballot(bad) != 0 ? __builtin_nanf("") : s;
}

// The codes of a block's four values: round(127 sqrt(x / scale)) and round(255 sqrt(sqrt(x / scale))), with every operation
// correctly rounded, so that they are what any implementation in this order gives.  Correctly rounded quotients and roots take
// ten instructions each and bound the kernel (250 M parameters: 1,026 us so, 705 as below), so they are computed
// from the hardware's reciprocal and root first (one unit in the last place each).  Those differ by less than 127 * 4e-7 and
// 255 * 5e-7 codes; only where a value lies that near the middle between two codes, twice as near for safety, the wave
// computes it the long way.
template <bool SECOND>
__device__ __forceinline__ void codes(const float (&x)[kPer], float scale, float (&q)[kPer]) {
  constexpr float kTop = SECOND ? 255.0f : 127.0f, kNear = SECOND ? 2.6e-4f : 1.1e-4f;
  const bool plain = scale > 1e-30f;  // (the reciprocal of less may not be finite; NaN takes the long way too)
  bool near = !plain;
  const float inv = __builtin_amdgcn_rcpf(plain ? scale : 1.0f);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    float r = __builtin_amdgcn_sqrtf(x[e] * inv);
    if (SECOND) r = __builtin_amdgcn_sqrtf(r);
    r *= kTop;
    q[e] = rintf(r);
    near |= fabsf(r - q[e]) > 0.5f - kNear;
  }
  if (__ballot(near) != 0) {
    const float by = scale > 0.0f ? scale : 1.0f;
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      float r = sqrtf(x[e] / by);
      if (SECOND) r = sqrtf(r);
      q[e] = rintf(r * kTop);
    }
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) q[e] = fminf(fmaxf(q[e], 0.0f), kTop);  // (NaN becomes 0)
}

// What the dither draws from: 24 bits for m and 24 for v, uniform and independent of each other, of the other elements' and of other
// keys' to what tests can tell.  Two and one rounds of xor-shifts and products; the factors are the fractions of the square roots
// of 2, 3 and 5 in 32 bits, made odd.
__device__ __forceinline__ uint32_t chance_m(int64_t i, uint32_t key) {
  uint32_t x = (static_cast<uint32_t>(i) + static_cast<uint32_t>(i >> 32) * 0x3c6ef373u) ^ key;
  x = (x ^ x >> 16) * 0x6a09e667u;
  x = (x ^ x >> 15) * 0xbb67ae85u;
  return x ^ x >> 16;
}
__device__ __forceinline__ uint32_t chance_v(uint32_t m) {
  m = (m ^ m >> 13) * 0x3c6ef373u;
  return m ^ m >> 16;
}
uint32_t dither_key(int64_t dither) {
  uint64_t x = static_cast<uint64_t>(dither) * 0x6a09e667f3bcc909u;
  x = (x ^ x >> 32) * 0xbb67ae8584caa73bu;
  return static_cast<uint32_t>(x ^ x >> 32);
}

// Codes rounded by chance: k is the one below x, and the one above it is taken with the probability (x - value(k)) / (value(k + 1)
// - value(k)).  The roots only choose k and need not be exact: next to a code's value either k gives that code almost surely.
template <bool SECOND>
__device__ __forceinline__ void dithered_codes(const float (&x)[kPer], float scale, const uint32_t (&chance)[kPer], float (&q)[kPer]) {
  constexpr float kTop = SECOND ? 255.0f : 127.0f, kAll = SECOND ? kTop * kTop * kTop * kTop : kTop * kTop;
  const bool plain = scale > 1e-30f;  // (as in codes(); the same in all lanes)
  const float by = scale > 0.0f ? scale : 1.0f, inv = __builtin_amdgcn_rcpf(plain ? scale : 1.0f);
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const float y = plain ? x[e] * inv : x[e] / by;
    float r = __builtin_amdgcn_sqrtf(y);
    if (SECOND) r = __builtin_amdgcn_sqrtf(r);
    const float k = floorf(fminf(kTop * r, kTop)), k1 = k + 1.0f;
    const float low = SECOND ? k * k * (k * k) : k * k, high = SECOND ? k1 * k1 * (k1 * k1) : k1 * k1;
    const float u = static_cast<float>(chance[e] >> 8) * 0x1p-24f;
    q[e] = k + (u * (high - low) < y * kAll - low ? 1.0f : 0.0f);
    q[e] = fminf(fmaxf(q[e], 0.0f), kTop);  // (NaN becomes 0)
  }
}

enum States { kBits32, kBits8, kBits8Dither };

template <class P, class G, bool MASTER, States STATES, bool STREAM>
__global__ __launch_bounds__(kAdamwThreads) void adamw_update_kernel(const UpdateTable t, const Scalars s,
                                                                     const float* __restrict__ coef) {
  constexpr bool BITS8 = STATES != kBits32;
  const int k = tensor_of(t.first, t.tensors, blockIdx.x);
  const Tensor& q = t.t[k];
  const int64_t count = q.count;
  const int64_t i = static_cast<int64_t>(static_cast<int>(blockIdx.x) - t.first[k]) * kChunk + threadIdx.x * kPer;
  const int n = static_cast<int>(max<int64_t>(0, min<int64_t>(kPer, count - i)));
  if (!BITS8 && n == 0) return;
  const float c = coef != nullptr ? *coef : 1.0f;
  float g[kPer], p[kPer], m[kPer], v[kPer];
  load4<STREAM>(static_cast<const G*>(q.grad) + i, n, g);
  if constexpr (MASTER) load4<STREAM>(q.master + i, n, p);
  else load4<STREAM>(static_cast<const P*>(q.param) + i, n, p);
  const int64_t block = i / PPO_ADAMW_BLOCK;
  if constexpr (BITS8) {
    const bool some = block * PPO_ADAMW_BLOCK < count;  // (of the wave's block)
    const float ms = some ? q.m_scale[block] : 0.0f, vs = some ? q.v_scale[block] : 0.0f;
    load4<STREAM>(static_cast<const int8_t*>(q.m) + i, n, m);
    load4<STREAM>(static_cast<const uint8_t*>(q.v) + i, n, v);
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      const float a = fabsf(m[e]) * (1.0f / 127.0f), b = v[e] * (1.0f / 255.0f);
      m[e] = (m[e] < 0.0f ? -ms : ms) * (a * a);
      const float b2 = b * b;
      v[e] = vs * (b2 * b2);
    }
  } else {
    load4<STREAM>(static_cast<const float*>(q.m) + i, n, m);
    load4<STREAM>(static_cast<const float*>(q.v) + i, n, v);
  }
#pragma unroll
  for (int e = 0; e < kPer; ++e) {
    const float d = g[e] * c;
    m[e] = m[e] + s.w1 * (d - m[e]);
    v[e] = v[e] * s.b2;
    v[e] = v[e] + (s.c2 * d) * d;
    p[e] = p[e] * q.decay;
    if (BITS8 && s.eps >= 1e-16f)  // beside the states' rounding the last bit of the step does not count
      p[e] = p[e] + (q.neg_step * m[e]) * __builtin_amdgcn_rcpf(__builtin_amdgcn_sqrtf(v[e]) * q.inv_bc2_sqrt + s.eps);
    else
      p[e] = p[e] + (q.neg_step * m[e]) / (sqrtf(v[e]) / q.bc2_sqrt + s.eps);
  }
  if constexpr (BITS8) {
    // elements past the end hold zeros: g, m and v
    float am[kPer];
#pragma unroll
    for (int e = 0; e < kPer; ++e) am[e] = fabsf(m[e]);
    const float ms = block_scale(am), vs = block_scale(v);
    float qm[kPer], qv[kPer];
    if constexpr (STATES == kBits8Dither) {
      uint32_t for_m[kPer], for_v[kPer];
#pragma unroll
      for (int e = 0; e < kPer; ++e) {
        for_m[e] = chance_m(i + e, q.key);
        for_v[e] = chance_v(for_m[e]);
      }
      dithered_codes<false>(am, ms, for_m, qm);
      dithered_codes<true>(v, vs, for_v, qv);
    } else {
      codes<false>(am, ms, qm);
      codes<true>(v, vs, qv);
    }
#pragma unroll
    for (int e = 0; e < kPer; ++e) {
      qm[e] = copysignf(qm[e], m[e]);
      if (v[e] > 0.0f) qv[e] = fmaxf(qv[e], 1.0f);
    }
    if (n == 0) return;
    store4<STREAM>(static_cast<int8_t*>(q.m) + i, n, qm);
    store4<STREAM>(static_cast<uint8_t*>(q.v) + i, n, qv);
    if (threadIdx.x % kWave == 0) {
      q.m_scale[block] = ms;
      q.v_scale[block] = vs;
    }
  } else {
    store4<STREAM>(static_cast<float*>(q.m) + i, n, m);
    store4<STREAM>(static_cast<float*>(q.v) + i, n, v);
  }
  if constexpr (MASTER) store4<STREAM>(q.master + i, n, p);
  store4<STREAM>(static_cast<P*>(q.param) + i, n, p);
}

int64_t chunks_of(const ppo_adamw_tensor& t) { return ceil_div(t.count, kChunk); }

// What a launch may hold: fewer than 2^32 threads.  Tensors that would make it more go to the next one.
constexpr int64_t kMaxCount = int64_t{1} << 33;  // of a tensor
constexpr int64_t kMaxChunks = (int64_t{1} << 32) / kAdamwThreads - 1;
static_assert(kMaxCount / kChunk <= kMaxChunks, "any tensor by itself fits a launch");
static_assert(kMaxGrads * (kMaxCount / kNormChunk) < INT32_MAX, "so do a norm launch's chunks a 32-bit index");

int64_t norm_partials(const ppo_adamw_tensor* tensors, int32_t count) {
  // a bound: each launch writes at most kNormBlocks, and there is one per kMaxGrads tensors of a type
  return static_cast<int64_t>(kNormBlocks) * (count / kMaxGrads + 2);
}

template <class P, class G, bool MASTER, States STATES>
void launch_states(bool stream, int chunks, hipStream_t st, const UpdateTable& t, const Scalars& s, const float* coef) {
  if (stream)
    hipLaunchKernelGGL((adamw_update_kernel<P, G, MASTER, STATES, true>), dim3(chunks), dim3(kAdamwThreads), 0, st, t, s, coef);
  else
    hipLaunchKernelGGL((adamw_update_kernel<P, G, MASTER, STATES, false>), dim3(chunks), dim3(kAdamwThreads), 0, st, t, s, coef);
}

template <class P, class G, bool MASTER>
void launch_update(States states, bool stream, int chunks, hipStream_t st, const UpdateTable& t, const Scalars& s, const float* coef) {
  if (states == kBits32) launch_states<P, G, MASTER, kBits32>(stream, chunks, st, t, s, coef);
  else if (states == kBits8) launch_states<P, G, MASTER, kBits8>(stream, chunks, st, t, s, coef);
  else launch_states<P, G, MASTER, kBits8Dither>(stream, chunks, st, t, s, coef);
}

// The kinds a launch holds together: bit 0 bf16 param, bit 1 bf16 gradient, bit 2 master, the rest the states.
constexpr int kKinds = 3 << 3;
int kind_of(const ppo_adamw_tensor& t) {
  const States states = t.state_bits == 32 ? kBits32 : t.dither == 0 ? kBits8 : kBits8Dither;
  return (t.param_type == PPO_TYPE_BF16 ? 1 : 0) | (t.grad_type == PPO_TYPE_BF16 ? 2 : 0) | (t.master != nullptr ? 4 : 0) | states << 3;
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_adamw_workspace_bytes(const ppo_adamw_tensor* tensors, int32_t count) {
  if (tensors == nullptr || count < 1) return 0;
  return 256 + sizeof(double) * static_cast<size_t>(norm_partials(tensors, count));
}

extern "C" int ppo_adamw_step(const ppo_adamw_tensor* tensors, int32_t count, double max_norm, double beta1, double beta2,
                              double eps, float* norm_out, void* workspace, size_t workspace_bytes,
                              ppo_stream_t stream) {
  PPO_REQUIRE(tensors != nullptr && count >= 1, "ppo_adamw_step: %d tensors", count);
  PPO_REQUIRE(beta1 >= 0.0 && beta1 < 1.0 && beta2 >= 0.0 && beta2 < 1.0 && eps >= 0.0, "ppo_adamw_step: beta1=%g beta2=%g eps=%g",
              beta1, beta2, eps);
  for (int i = 0; i < count; ++i) {
    const ppo_adamw_tensor& t = tensors[i];
    PPO_REQUIRE(t.count >= 0 && t.count < kMaxCount, "ppo_adamw_step: tensor %d holds %lld elements", i, (long long)t.count);
    PPO_REQUIRE((t.param_type == PPO_TYPE_F32 || t.param_type == PPO_TYPE_BF16) &&
                    (t.grad_type == PPO_TYPE_F32 || t.grad_type == PPO_TYPE_BF16),
                "ppo_adamw_step: tensor %d: param_type=%d grad_type=%d", i, t.param_type, t.grad_type);
    PPO_REQUIRE(t.bc1 > 0.0 && t.bc2_sqrt > 0.0, "ppo_adamw_step: tensor %d: bias corrections must be positive", i);
    PPO_REQUIRE(t.state_bits == 32 || t.state_bits == 8, "ppo_adamw_step: tensor %d: state_bits=%d", i, t.state_bits);
    PPO_REQUIRE(t.master == nullptr || t.param_type == PPO_TYPE_BF16, "ppo_adamw_step: tensor %d: a master of an fp32 param", i);
    PPO_REQUIRE(t.param_type == PPO_TYPE_BF16 || t.grad_type == PPO_TYPE_F32, "ppo_adamw_step: tensor %d: a bf16 gradient of an fp32 param", i);
    PPO_REQUIRE(t.count == 0 || (t.param && t.grad && t.exp_avg && t.exp_avg_sq &&
                                 (t.state_bits == 32 || (t.m_scale && t.v_scale))),
                "ppo_adamw_step: tensor %d: null pointer", i);
    PPO_REQUIRE(reinterpret_cast<uintptr_t>(t.param) % type_size(t.param_type) == 0 &&
                    reinterpret_cast<uintptr_t>(t.grad) % type_size(t.grad_type) == 0 &&
                    reinterpret_cast<uintptr_t>(t.master) % 4 == 0 && reinterpret_cast<uintptr_t>(t.m_scale) % 4 == 0 &&
                    reinterpret_cast<uintptr_t>(t.v_scale) % 4 == 0 &&
                    (t.state_bits == 8 || (reinterpret_cast<uintptr_t>(t.exp_avg) % 4 == 0 &&
                                           reinterpret_cast<uintptr_t>(t.exp_avg_sq) % 4 == 0)),
                "ppo_adamw_step: tensor %d: pointers must be aligned to their elements", i);
  }
  const bool norm = max_norm > 0.0 || norm_out != nullptr;
  const size_t need = ppo_adamw_workspace_bytes(tensors, count);
  PPO_REQUIRE(!norm || (workspace != nullptr && workspace_bytes >= need), "ppo_adamw_step: workspace too small (%zu < %zu)",
              workspace_bytes, need);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 8 == 0, "ppo_adamw_step: the workspace must be 8-byte aligned");
  hipStream_t st = static_cast<hipStream_t>(stream);
  float* coef = nullptr;
  if (norm) {
    coef = static_cast<float*>(workspace);
    double* partial = reinterpret_cast<double*>(static_cast<char*>(workspace) + 256);
    int partials = 0;
    for (int type : {PPO_TYPE_F32, PPO_TYPE_BF16}) {
      int i = 0;
      while (i < count) {
        NormTable t{};
        int64_t chunks = 0;
        for (; i < count && t.tensors < kMaxGrads; ++i) {
          if (tensors[i].grad_type != type || tensors[i].count == 0) continue;
          t.grad[t.tensors] = tensors[i].grad;
          t.count[t.tensors] = tensors[i].count;
          t.first[t.tensors++] = static_cast<int32_t>(chunks);
          chunks += ceil_div(tensors[i].count, kNormChunk);
        }
        if (t.tensors == 0) break;
        t.first[t.tensors] = static_cast<int32_t>(chunks);
        const int blocks = static_cast<int>(std::min<int64_t>(chunks, kNormBlocks));
        if (type == PPO_TYPE_F32)
          hipLaunchKernelGGL(adamw_norm_kernel<float>, dim3(blocks), dim3(kAdamwThreads), 0, st, t, static_cast<int>(chunks), partial + partials);
        else
          hipLaunchKernelGGL(adamw_norm_kernel<__bf16>, dim3(blocks), dim3(kAdamwThreads), 0, st, t, static_cast<int>(chunks), partial + partials);
        if (int rc = check_launch("adamw_norm_kernel")) return rc;
        partials += blocks;
      }
    }
    hipLaunchKernelGGL(adamw_clip_kernel, dim3(1), dim3(kAdamwThreads), 0, st, partial, partials, static_cast<float>(max_norm), coef, norm_out);
    if (int rc = check_launch("adamw_clip_kernel")) return rc;
  }
  const Scalars s{static_cast<float>(1.0 - beta1), static_cast<float>(beta2), static_cast<float>(1.0 - beta2),
                  static_cast<float>(eps)};
  int64_t bytes = 0;
  for (int i = 0; i < count; ++i) {
    const ppo_adamw_tensor& t = tensors[i];
    bytes += t.count * (type_size(t.param_type) + type_size(t.grad_type) + (t.master ? 4 : 0) + (t.state_bits == 8 ? 2 : 8));
  }
  const bool past_cache = bytes > kCacheBytes;
  for (int kind = 0; kind < kKinds; ++kind) {
    int i = 0;
    while (i < count) {
      UpdateTable t{};
      int64_t chunks = 0;
      for (; i < count && t.tensors < kMaxTensors; ++i) {
        const ppo_adamw_tensor& a = tensors[i];
        if (kind_of(a) != kind || a.count == 0) continue;
        if (chunks + chunks_of(a) > kMaxChunks) break;
        Tensor& b = t.t[t.tensors];
        b = Tensor{a.param, a.grad, a.master, a.exp_avg, a.exp_avg_sq, a.m_scale, a.v_scale, a.count,
                   static_cast<float>(-(a.lr / a.bc1)), static_cast<float>(1.0 - a.lr * a.weight_decay),
                   static_cast<float>(a.bc2_sqrt), static_cast<float>(1.0 / a.bc2_sqrt), dither_key(a.dither)};
        t.first[t.tensors++] = static_cast<int32_t>(chunks);
        chunks += chunks_of(a);
      }
      if (t.tensors == 0) break;
      t.first[t.tensors] = static_cast<int32_t>(chunks);
      const States states = static_cast<States>(kind >> 3);
      switch (kind & 7) {
        case 0: launch_update<float, float, false>(states, past_cache, static_cast<int>(chunks), st, t, s, coef); break;
        case 1: launch_update<__bf16, float, false>(states, past_cache, static_cast<int>(chunks), st, t, s, coef); break;
        case 3: launch_update<__bf16, __bf16, false>(states, past_cache, static_cast<int>(chunks), st, t, s, coef); break;
        case 5: launch_update<__bf16, float, true>(states, past_cache, static_cast<int>(chunks), st, t, s, coef); break;
        case 7: launch_update<__bf16, __bf16, true>(states, past_cache, static_cast<int>(chunks), st, t, s, coef); break;
        default: return fail(PPO_EINVAL, "ppo_adamw_step: kind %d", kind);
      }
      if (int rc = check_launch("adamw_update_kernel")) return rc;
    }
  }
  return PPO_OK;
}
