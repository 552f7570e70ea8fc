// Token log-probabilities and the clipped policy loss with a KL term, forward and gradient (ppo_token_log_probs,
// ppo_token_ppo_loss): the categorical counterpart of loss.hip's Gaussian head.
//
// With c = log2(e) / temperature, m = max_j x_j and t_j = c (x_j - m):
//   S = sum_j 2^t_j,  E = sum_j 2^t_j t_j,  lp = ln2 (t_token - log2 S),  H = ln2 (log2 S - E / S),
//   d_logits_j = 2^t_j (A + B t_j) + [j = token] g k,
//   k = 1 / (N temperature),  B = k entropy_coef ln2 / S,  A = k (entropy_coef H - g) / S - B log2 S
// (p_j = 2^t_j / S and log p_j = ln2 (t_j - log2 S) put into the header's formula).  The difference comes first: next to the
// maximum it is exact, however far from zero the row lies.  As one fused multiply-add, c x_j - (c m), t_j would carry the rounding
// of c m, half an ulp of it and another one for each part's m: rows at 1e4 were 3e-4 off, rows masked by -1e10 not finite.
// A logit of -inf has 2^t = 0 exactly; where t itself is a factor it is raised to kFloor, 2^kFloor being 0 too, so that 0 t
// stays 0.
//
// Bound by memory: the logits once in, their gradient once out.  So a row is read once and stays in registers between its
// sums and its gradient (token_row_kernel); only rows too wide for that are read twice (token_wide_kernel).  Each wave
// takes its own maximum and sums, and the waves' (m, S, E) are joined after the one barrier of a row.
// 8,192 x 131,072 bf16, a quarter of the rows masked: 720 us a call, 5.2 TB/s; log-probabilities of 8,192 x 32,000: 73 us
// (715 and 70 with the fused multiply-add above).
#include "elem.hpp"

namespace ppo {
namespace {

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1000.0f;
// sums over rows per row: s, k, H, clipped, old_logp - lp, counts, (2 unused)
constexpr int kTerms = 6, kTermStride = 8;
constexpr int kCountRows = 512;  // up to so many rows each block counts them itself (us so -> by a launch of its own: 128 x 32,000 bf16
                                 // 14.4 -> 15.6, 512 20.8 -> 21.8, 1,024 33.2 -> 31.5, 4,096 125 -> 113)
constexpr int kCountThreads = 1024;

struct LossKernelArgs {
  ppo_token_loss_args a;
  float* inv_n;   // 1 / N of token_count_kernel, where that ran
  float* terms;   // [rows][kTermStride]
  bool stream;    // (kCacheBytes)
  int32_t count;  // 1: the block counts the rows, 2: inv_n holds 1 / N, 0: given_inv_n does
  float given_inv_n;
  float c, inv_temp, clip_lo, clip_hi, kl_coef, entropy_coef;
};

__device__ __forceinline__ bool row_counts(const ppo_token_loss_args& a, int64_t r, int64_t& tok) {
  tok = -1;
  if (a.mask != nullptr && a.mask[r] == 0) return false;
  tok = token_at(a.tokens, a.token_type, r, a.vocab);
  return tok >= 0;
}

// A block per row, kGridRows of them along x, more along y: a launch may not hold 2^32 threads along one axis, which 4,194,304
// blocks of 1,024 would.
constexpr int64_t kGridRows = 1 << 20;
dim3 row_grid(int64_t rows) {
  return dim3(static_cast<uint32_t>(std::min(rows, kGridRows)), static_cast<uint32_t>(ceil_div(rows, kGridRows)));
}
__device__ __forceinline__ int64_t block_row() { return blockIdx.x + static_cast<int64_t>(blockIdx.y) * kGridRows; }

template <class R>
__device__ __forceinline__ R wave_sum(R x) {
  for (int d = kWave / 2; d > 0; d >>= 1) x += __shfl_xor(x, d, kWave);
  return x;
}

__device__ __forceinline__ float wave_max(float x) {
  for (int d = kWave / 2; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor(x, d, kWave));
  return x;
}

__device__ __forceinline__ int32_t rows_counted(const LossKernelArgs& q, int first, int step) {
  int32_t n = 0;
  for (int64_t r = first; r < q.a.rows; r += 4 * step) {
    bool in[4];  // four rows' loads in flight
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int64_t i = min(r + u * step, q.a.rows - 1);
      const bool kept = q.a.mask == nullptr || q.a.mask[i] != 0;
      in[u] = (token_at(q.a.tokens, q.a.token_type, i, q.a.vocab) >= 0) & kept & (r + u * step < q.a.rows);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) n += in[u] ? 1 : 0;
  }
  return n;
}

__global__ __launch_bounds__(kCountThreads) void token_count_kernel(const LossKernelArgs q) {
  __shared__ int32_t part[kCountThreads / kWave];
  const int32_t n = wave_sum(rows_counted(q, threadIdx.x, kCountThreads));
  if (threadIdx.x % kWave == 0) part[threadIdx.x / kWave] = n;
  __syncthreads();
  if (threadIdx.x == 0) {
    int32_t all = 0;
    for (int w = 0; w < kCountThreads / kWave; ++w) all += part[w];
    *q.inv_n = all > 0 ? static_cast<float>(1.0 / all) : 0.0f;
  }
}

struct RowSums {
  float m, s, e;
};

// The sums of one part of a row next to those of another.
__device__ __forceinline__ RowSums join(const RowSums& u, const RowSums& v, float c) {
#pragma clang fp contract(off)
  RowSums o;  // (no fused multiply-add: the same bits whichever part comes first)
  o.m = fmaxf(u.m, v.m);
  const float du = u.m == o.m ? 0.0f : fmaxf((u.m - o.m) * c, kFloor), dv = v.m == o.m ? 0.0f : fmaxf((v.m - o.m) * c, kFloor);
  const float fu = __builtin_amdgcn_exp2f(du), fv = __builtin_amdgcn_exp2f(dv);
  o.s = u.s * fu + v.s * fv;
  o.e = (u.e + u.s * du) * fu + (v.e + v.s * dv) * fv;
  return o;
}

__device__ __forceinline__ RowSums join_lanes(const RowSums& u, int d, float c) {
  return join(u, RowSums{__shfl_xor(u.m, d, kWave), __shfl_xor(u.s, d, kWave), __shfl_xor(u.e, d, kWave)}, c);
}

template <int WAVES>
struct RowShared {
  RowSums sums[WAVES];
  int32_t count[WAVES];
};

// What a row contributes: logp, H, log2 S, the derivative g by logp, and the terms of the means.
struct RowTerms {
  float lp, h, log2_s, g;
  float term[kTerms];
  bool live;  // (nothing but -inf: no distribution; a NaN goes on)
};

// k = exp(d) - d - 1, never negative, grown = exp(d) - 1.  Near the reference policy k is d^2 / 2, far below the ones that exp(d) - 1
// is made of, and below the last bit of `grown` too: there its series, whose first term left out is 1.2e-8 of it at the end.
__device__ __forceinline__ float kl_of(float d, float grown) {
  if (!(fabsf(d) < 0.25f)) return grown - d;
  return d * d * (0.5f + d * (1.0f / 6 + d * (1.0f / 24 + d * (1.0f / 120 + d * (1.0f / 720 + d * (1.0f / 5040))))));
}

template <bool LOSS>
__device__ __forceinline__ RowTerms row_terms(const LossKernelArgs& q, int64_t r, const RowSums& sums, float x_tok) {
  RowTerms o{};
  o.term[5] = 1.0f;
  o.live = sums.m > -INFINITY || sums.s != sums.s;
  if (!o.live) return o;
  o.log2_s = log2f(sums.s);
  o.lp = kLn2 * ((x_tok - sums.m) * q.c - o.log2_s);
  o.h = kLn2 * (o.log2_s - sums.e / sums.s);
  if (!LOSS) return o;
  const float old = q.a.old_logp[r], adv = q.a.advantages[r];
  const float ratio = expf(o.lp - old);
  const float clipped = fminf(fmaxf(ratio, q.clip_lo), q.clip_hi);
  const float first = -adv * ratio, second = -adv * clipped;
  o.g = first >= second ? first : first < second ? 0.0f : first + second;  // (NaN goes on)
  o.term[0] = first != first || second != second ? first + second : fmaxf(first, second);
  if (q.a.ref_logp != nullptr) {
    const float d = q.a.ref_logp[r] - o.lp, grown = expm1f(d);
    o.term[1] = kl_of(d, grown);
    if (q.kl_coef != 0.0f) o.g -= q.kl_coef * grown;  // (0: k is only reported, and may be infinite)
  }
  o.term[2] = o.h;
  o.term[3] = ratio != clipped ? 1.0f : 0.0f;
  o.term[4] = old - o.lp;
  return o;
}

// What its gradient needs: t = (x - m) c, d = 2^t (a + b t), + at at the token.
struct RowCoefs {
  float c, m, a, b, at;
  bool live;
};

// Joins the waves' sums (the row's only barrier) and writes logp, entropy and the loss terms.
template <int NT, bool LOSS>
__device__ __forceinline__ RowCoefs finish_row(const LossKernelArgs& q, int64_t r, RowSums mine, float x_tok, int32_t counted,
                                               RowShared<NT / kWave>& sh, bool write) {
  constexpr int WAVES = NT / kWave;
  if constexpr (WAVES > 1) {
    if (threadIdx.x % kWave == 0) {
      sh.sums[threadIdx.x / kWave] = mine;
      if (LOSS) sh.count[threadIdx.x / kWave] = counted;
    }
    __syncthreads();
    mine = sh.sums[threadIdx.x % WAVES];
    counted = LOSS ? sh.count[threadIdx.x % WAVES] : 0;
#pragma unroll
    for (int d = WAVES / 2; d > 0; d >>= 1) {
      mine = join_lanes(mine, d, q.c);
      if (LOSS) counted += __shfl_xor(counted, d, kWave);
    }
  }
  const RowTerms u = row_terms<LOSS>(q, r, mine, x_tok);
  if (write) {
    if (q.a.logp != nullptr) q.a.logp[r] = u.lp;
    if (q.a.entropy != nullptr) q.a.entropy[r] = u.h;
    if (LOSS)
#pragma unroll
      for (int i = 0; i < kTerms; ++i) q.terms[r * kTermStride + i] = u.term[i];
  }
  RowCoefs o{q.c, mine.m, 0.0f, 0.0f, 0.0f, u.live};
  if (LOSS && u.live) {
    const float inv_n = q.count == 1 ? 1.0f / static_cast<float>(counted) : q.count == 2 ? *q.inv_n : q.given_inv_n;
    const float k = inv_n * q.inv_temp, inv_s = 1.0f / mine.s;
    o.b = k * q.entropy_coef * kLn2 * inv_s;
    o.a = k * (q.entropy_coef * u.h - u.g) * inv_s - o.b * u.log2_s;
    o.at = k * u.g;
  }
  return o;
}

// A row that does not count, or has no distribution: its gradient is zero.
template <class T, int NT>
__device__ __forceinline__ void zero_gradient(T* dx, int64_t first, int64_t vocab) {
  constexpr int V = kVec<T>;
  const float zero[V] = {};
  for (int64_t j = first + threadIdx.x * V; j < vocab; j += NT * V) {
    if (j + V <= vocab) store_piece(dx + j, zero);
    else
      for (int64_t i = j; i < vocab; ++i) dx[i] = static_cast<T>(0.0f);
  }
}

template <bool LOSS>
__device__ __forceinline__ void skip_row(const LossKernelArgs& q, int64_t r) {
  if (threadIdx.x != 0) return;
  if (q.a.logp != nullptr) q.a.logp[r] = 0.0f;
  if (q.a.entropy != nullptr) q.a.entropy[r] = 0.0f;
  if (LOSS)
    for (int i = 0; i < kTerms; ++i) q.terms[r * kTermStride + i] = 0.0f;
}

__device__ __forceinline__ float gradient_of(float x, const RowCoefs& o) {
  const float t = fmaxf((x - o.m) * o.c, kFloor);
  return __builtin_amdgcn_exp2f(t) * fmaf(o.b, t, o.a);
}

// 16-byte pieces of a row in the registers of NT threads, K each: piece k of thread i holds the columns from
// first + (k NT + i) V on (vocab >= V).  The last piece of a row whose width is no multiple of V is read from V columns before
// the end; what it shares with the piece before it, and pieces past the end, become -inf, which adds nothing to a sum.
template <class T, int NT, int K>
struct RowPieces {
  static constexpr int V = kVec<T>;
  RawPiece raw[K];
  int vocab, first, tid, wave;

  __device__ __forceinline__ RowPieces(int vocab_, int first_) : vocab(vocab_), first(first_), tid(threadIdx.x) {
    wave = __builtin_amdgcn_readfirstlane(tid / kWave * kWave);
  }
  __device__ __forceinline__ int column(int k) const { return first + (k * NT + tid) * V; }
  // whether the wave's pieces lie inside the row, partly or not at all: the same for its lanes
  __device__ __forceinline__ bool whole(int k) const { return first + (k * NT + wave + kWave) * V <= vocab; }
  __device__ __forceinline__ bool some(int k) const { return first + (k * NT + wave) * V < vocab; }
  __device__ __forceinline__ uint32_t offset(int j) const { return static_cast<uint32_t>(j) * static_cast<uint32_t>(sizeof(T)); }

  template <bool STREAM>
  __device__ __forceinline__ void load(const T* x) {
#pragma unroll
    for (int k = 0; k < K; ++k)  // a uniform base and 32 bits of offset
      raw[k] = load_raw<STREAM>(reinterpret_cast<const T*>(reinterpret_cast<const char*>(x) + offset(min(column(k), vocab - V))));
  }

  // The wave's maximum and sums.
  __device__ __forceinline__ RowSums sums(float c) {
    RowSums mine{-INFINITY, 0.0f, 0.0f};
    forget(tid);  // (columns are computed again where they are needed, not kept)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (!whole(k)) {
        const int skip = column(k) - min(column(k), vocab - V);
#pragma unroll
        for (int e = 0; e < V; ++e)
          if (e < skip) make_neg_inf<T>(raw[k], e);
      }
#pragma unroll
      for (int e = 0; e < V; ++e) mine.m = fmaxf(mine.m, element<T>(raw[k], e));
      forget(raw[k], mine.m);
      __builtin_amdgcn_sched_barrier(0);  // one piece at a time: its converted values are gone before the next one's
    }
    mine.m = wave_max(mine.m);
    const float m = mine.m > -INFINITY ? mine.m : 0.0f;  // (nothing but -inf: sums of 0)
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (some(k)) {
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float t = (element<T>(raw[k], e) - m) * c, p = __builtin_amdgcn_exp2f(t);
          mine.s += p;
          mine.e = fmaf(p, fmaxf(t, kFloor), mine.e);
        }
      }
      forget(raw[k], mine.s);
      __builtin_amdgcn_sched_barrier(0);
    }
    mine.s = wave_sum(mine.s);
    mine.e = wave_sum(mine.e);
    return mine;
  }

  __device__ __forceinline__ void gradient(T* dx, int tok, const RowCoefs& o, bool stream) {
    forget(tid);
#pragma unroll
    for (int k = 0; k < K; ++k) {
      if (some(k)) {
        const int at = min(column(k), vocab - V);
        float d[V];
#pragma unroll
        for (int e = 0; e < V; ++e) d[e] = gradient_of(element<T>(raw[k], e), o);
        const uint32_t hit = static_cast<uint32_t>(tok - at);
        if (hit < V)
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (static_cast<uint32_t>(e) == hit) d[e] += o.at;
        if (whole(k)) {
          T* to = reinterpret_cast<T*>(reinterpret_cast<char*>(dx) + offset(at));
          if (stream) store_piece<true>(to, d);
          else store_piece(to, d);
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (e >= column(k) - at) dx[at + e] = static_cast<T>(d[e]);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
  }
};

// One block of NT threads per row, the whole row in its registers (NT K V >= vocab).
template <class T, int NT, int K, bool LOSS>
__global__ __launch_bounds__(NT, NT == 512 ? 4 : 1) void token_row_kernel(const LossKernelArgs q) {
  __shared__ RowShared<NT / kWave> sh;
  const ppo_token_loss_args& a = q.a;
  const int64_t r = block_row();
  if (r >= a.rows) return;
  const int vocab = static_cast<int>(a.vocab);
  const T* x = static_cast<const T*>(a.logits) + r * a.ld_logits;
  T* dx = LOSS && a.d_logits != nullptr ? static_cast<T*>(a.d_logits) + r * a.ld_d_logits : nullptr;
  int64_t tok;
  if (!row_counts(a, r, tok)) {
    skip_row<LOSS>(q, r);
    if (dx != nullptr) zero_gradient<T, NT>(dx, 0, vocab);
    return;
  }
  RowPieces<T, NT, K> row(vocab, 0);
  if (q.stream) row.template load<true>(x);
  else row.template load<false>(x);
  float x_tok = static_cast<float>(x[tok]);
  const int32_t counted = LOSS && q.count == 1 ? wave_sum(rows_counted(q, threadIdx.x, NT)) : 0;
  const RowSums mine = row.sums(q.c);
  arrived(x_tok);
  const RowCoefs o = finish_row<NT, LOSS>(q, r, mine, x_tok, counted, sh, threadIdx.x == 0);
  if (dx == nullptr) return;
  if (o.live) row.gradient(dx, static_cast<int>(tok), o, q.stream);
  else zero_gradient<T, NT>(dx, 0, vocab);
}

// The means from their sums; the same lane of the first wave holds the sum of the same term.
__device__ __forceinline__ void write_stats(const LossKernelArgs& q, double sum) {
  const double rows = __shfl(sum, 5, kWave), n = q.a.denom > 0.0 ? q.a.denom : rows, inv = rows > 0.0 ? 1.0 / n : 0.0;
  const double s = __shfl(sum, 0, kWave), k = __shfl(sum, 1, kWave), h = __shfl(sum, 2, kWave);
  if (threadIdx.x < 5) q.a.stats[1 + threadIdx.x] = static_cast<float>(sum * inv);
  if (threadIdx.x == 5) q.a.stats[0] = static_cast<float>((s + (q.a.kl_coef != 0.0 ? q.a.kl_coef * k : 0.0) - q.a.entropy_coef * h) * inv);
  if (threadIdx.x == 6) q.a.stats[6] = static_cast<float>(n);
  if (threadIdx.x == 7) q.a.stats[7] = 0.0f;
}

// The means over rows, fp64 sums in a fixed order.
template <int NT>
__global__ __launch_bounds__(NT) void token_stats_kernel(const LossKernelArgs q) {
  constexpr int WAVES = NT / kWave;
  __shared__ double part[kTerms][WAVES];
  double sum[kTerms] = {};
#pragma unroll 4
  for (int64_t r = threadIdx.x; r < q.a.rows; r += NT) {
    const float4* t = reinterpret_cast<const float4*>(q.terms + r * kTermStride);
    const float4 u = t[0], v = t[1];
    sum[0] += u.x, sum[1] += u.y, sum[2] += u.z, sum[3] += u.w, sum[4] += v.x, sum[5] += v.y;
  }
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < kTerms; ++i) sum[i] += __shfl_xor(sum[i], d, kWave);
  if (threadIdx.x % kWave == 0)
#pragma unroll
    for (int i = 0; i < kTerms; ++i) part[i][threadIdx.x / kWave] = sum[i];
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  double all = 0.0;  // lane i: term i
  if (threadIdx.x < kTerms)
#pragma unroll
    for (int w = 0; w < WAVES; ++w) all += part[threadIdx.x][w];
  write_stats(q, all);
}

// A few wide rows, which one compute unit each would leave waiting for its arithmetic: a row is cut into parts of
// kPartThreads kPartPieces pieces, a block each.  token_part_kernel leaves a part's sums; then token_joined_kernel's one wave
// per row joins them, or each block of token_part_gradient_kernel does before it reads its part again, and one more block the
// means of all rows.  Worth it (us, in one kernel -> in parts) for the loss of rows from 16,384 logits on (in a graph: 16 x 16,384
// bf16 9.2 -> 8.0, 64 x 16,384 fp32 10.4 -> 7.9, 16 x 32,000 bf16 12.3 -> 8.2, 8 x 131,072 23.2 -> 8.0, 64 x 131,072 26.0 ->
// 14.9), up to kSplitLossRows, since the block of the means has a lane for each row (more rows are not measured), and for
// log-probabilities of up to kSplitRows from 65,536 on (8 x 131,072 bf16 10.8 -> 9.3, 257 23.3 -> 16.2, 512 fp32 42.8 -> 43.0; 8 x 50,021 8.5 -> 9.4).
constexpr int kPartThreads = 256, kPartPieces = 4, kMaxParts = kWave;
constexpr int64_t kSplitRows = 256, kSplitVocab = 65536, kSplitLossRows = kWave, kSplitLossVocab = 16384;

struct RowPart {
  RowSums sums;
  float x_tok;  // of part 0 (d_logits may be the logits, so nobody reads it later)
};

template <class T>
__global__ __launch_bounds__(kPartThreads) void token_part_kernel(const LossKernelArgs q, RowPart* __restrict__ parts) {
  __shared__ RowSums sh[kPartThreads / kWave];
  const ppo_token_loss_args& a = q.a;
  const int64_t r = blockIdx.y;
  int64_t tok;
  if (!row_counts(a, r, tok)) return;
  const T* x = static_cast<const T*>(a.logits) + r * a.ld_logits;
  RowPieces<T, kPartThreads, kPartPieces> row(static_cast<int>(a.vocab), blockIdx.x * (kPartThreads * kPartPieces * kVec<T>));
  row.template load<false>(x);
  const float x_tok = blockIdx.x == 0 ? static_cast<float>(x[tok]) : 0.0f;
  RowSums mine = row.sums(q.c);
  if (threadIdx.x % kWave == 0) sh[threadIdx.x / kWave] = mine;
  __syncthreads();
  if (threadIdx.x >= kWave) return;
  mine = sh[threadIdx.x % (kPartThreads / kWave)];
#pragma unroll
  for (int d = kPartThreads / kWave / 2; d > 0; d >>= 1) mine = join_lanes(mine, d, q.c);
  if (threadIdx.x == 0) parts[r * gridDim.x + blockIdx.x] = RowPart{mine, x_tok};
}

// The parts of a row joined, in every lane.
__device__ __forceinline__ RowSums join_parts(const RowPart* parts, int n, float c) {
  const int lane = threadIdx.x % kWave;
  RowSums mine = lane < n ? parts[lane].sums : RowSums{-INFINITY, 0.0f, 0.0f};
#pragma unroll
  for (int d = kWave / 2; d > 0; d >>= 1) mine = join_lanes(mine, d, c);
  return mine;
}

__global__ __launch_bounds__(kWave) void token_joined_kernel(const LossKernelArgs q, const RowPart* __restrict__ parts, int n) {
  __shared__ RowShared<1> sh;
  const int64_t r = blockIdx.x;
  int64_t tok;
  if (!row_counts(q.a, r, tok)) {
    skip_row<false>(q, r);
    return;
  }
  finish_row<kWave, false>(q, r, join_parts(parts + r * n, n, q.c), parts[r * n].x_tok, 0, sh, threadIdx.x == 0);
}

// The same in one lane, in the same order and so with the same bits: join_parts joins the parts half a wave apart first, neighbours
// last, which is neighbours first where the parts come by their index' bits reversed.  Eight at a time, whose loads are in flight
// together (one after another the loss of 8 x 131,072 bf16 took 11.4 us, 8.2 so); have[l] waits for the other half of 16 << l
// parts.  join is the same either way round, and a part past the end changes nothing.
__device__ __forceinline__ RowSums join_parts_alone(const RowPart* parts, int n, float c) {
  constexpr int kLevels = 3;
  static_assert(8 << kLevels == kMaxParts, "a level for each halving of the parts");
  RowSums have[kLevels], x[8];
  int log_n = 3;
  while ((1 << log_n) < n) ++log_n;
  for (uint32_t k = 0; k < 1u << (log_n - 3); ++k) {
#pragma unroll
    for (int u = 0; u < 8; ++u) {
      const int i = static_cast<int>(__brev(8 * k + u) >> (32 - log_n));
      x[u] = parts[min(i, n - 1)].sums;
      if (i >= n) x[u] = RowSums{-INFINITY, 0.0f, 0.0f};
    }
#pragma unroll
    for (int w = 1; w < 8; w *= 2)
#pragma unroll
      for (int u = 0; u < 8; u += 2 * w) x[u] = join(x[u], x[u + w], c);
#pragma unroll
    for (int l = 0; l < kLevels; ++l) {
      if ((k >> l & 1) == 0) {
        have[l] = x[0];
        break;
      }
      x[0] = join(have[l], x[0], c);
    }
  }
  return x[0];
}

// The means, a lane per row (rows <= kSplitLossRows).
__device__ __forceinline__ void part_stats(const LossKernelArgs& q, const RowPart* parts, int n) {
  const int64_t r = threadIdx.x;
  int64_t tok;
  RowTerms u{};
  if (r < q.a.rows && row_counts(q.a, r, tok)) {
    const RowPart* row = parts + r * n;
    u = row_terms<true>(q, r, join_parts_alone(row, n, q.c), row[0].x_tok);
  }
  double mine = 0.0;  // lane i: term i
#pragma unroll
  for (int i = 0; i < kTerms; ++i) {
    const double x = wave_sum(static_cast<double>(u.term[i]));
    if (static_cast<int>(threadIdx.x) == i) mine = x;
  }
  write_stats(q, mine);
}

template <class T>
__global__ __launch_bounds__(kPartThreads) void token_part_gradient_kernel(const LossKernelArgs q, const RowPart* __restrict__ parts) {
  constexpr int kPart = kPartThreads * kPartPieces * kVec<T>;
  __shared__ RowShared<1> sh;
  const ppo_token_loss_args& a = q.a;
  const int64_t r = blockIdx.y;
  const int vocab = static_cast<int>(a.vocab), first = blockIdx.x * kPart, n = gridDim.x;
  if (r == a.rows) {
    if (first == 0 && threadIdx.x < kWave) part_stats(q, parts, n);
    return;
  }
  const T* x = static_cast<const T*>(a.logits) + r * a.ld_logits;
  T* dx = a.d_logits != nullptr ? static_cast<T*>(a.d_logits) + r * a.ld_d_logits : nullptr;
  if (dx == nullptr && first > 0) return;
  int64_t tok;
  if (!row_counts(a, r, tok)) {
    if (first == 0) skip_row<true>(q, r);
    if (dx != nullptr) zero_gradient<T, kPartThreads>(dx, first, min(first + kPart, vocab));
    return;
  }
  RowPieces<T, kPartThreads, kPartPieces> row(vocab, first);
  if (dx != nullptr) row.template load<false>(x);
  const int32_t counted = q.count == 1 ? wave_sum(rows_counted(q, threadIdx.x % kWave, kWave)) : 0;
  const RowCoefs o = finish_row<kWave, true>(q, r, join_parts(parts + r * n, n, q.c), parts[r * n].x_tok, counted, sh,
                                             first == 0 && threadIdx.x == 0);
  if (dx == nullptr) return;
  if (o.live) row.gradient(dx, static_cast<int>(tok), o, false);
  else zero_gradient<T, kPartThreads>(dx, first, min(first + kPart, vocab));
}

// Rows of any width: the sums in one pass, each thread rescaling its own when its maximum grows, the gradient in another.
constexpr int kWideThreads = 1024;

template <class T, bool LOSS>
__global__ __launch_bounds__(kWideThreads) void token_wide_kernel(const LossKernelArgs q) {
  constexpr int V = kVec<T>, NT = kWideThreads;
  __shared__ RowShared<NT / kWave> sh;
  const ppo_token_loss_args& a = q.a;
  const int64_t r = block_row();
  if (r >= a.rows) return;
  const T* x = static_cast<const T*>(a.logits) + r * a.ld_logits;
  T* dx = LOSS && a.d_logits != nullptr ? static_cast<T*>(a.d_logits) + r * a.ld_d_logits : nullptr;
  int64_t tok;
  if (!row_counts(a, r, tok)) {
    skip_row<LOSS>(q, r);
    if (dx != nullptr) zero_gradient<T, NT>(dx, 0, a.vocab);
    return;
  }
  auto load = [&](int64_t j, float (&v)[V]) {
    if (j + V <= a.vocab) {
      const auto p = load_piece(x + j);
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = static_cast<float>(p[e]);
    } else {
#pragma unroll
      for (int e = 0; e < V; ++e) v[e] = j + e < a.vocab ? static_cast<float>(x[j + e]) : -INFINITY;
    }
  };
  float x_tok = static_cast<float>(x[tok]);
  const int32_t counted = LOSS && q.count == 1 ? wave_sum(rows_counted(q, threadIdx.x, NT)) : 0;
  RowSums mine{-INFINITY, 0.0f, 0.0f};
  for (int64_t j = threadIdx.x * V; j < a.vocab; j += NT * V) {
    float v[V];
    load(j, v);
    RowSums part{-INFINITY, 0.0f, 0.0f};
#pragma unroll
    for (int e = 0; e < V; ++e) part.m = fmaxf(part.m, v[e]);
    const float m = fmaxf(part.m, mine.m);
    if (m > mine.m) mine = join(mine, RowSums{m, 0.0f, 0.0f}, q.c);
    const float from = m > -INFINITY ? m : 0.0f;
#pragma unroll
    for (int e = 0; e < V; ++e) {
      const float t = (v[e] - from) * q.c, p = __builtin_amdgcn_exp2f(t);
      mine.s += p;
      mine.e = fmaf(p, fmaxf(t, kFloor), mine.e);
    }
  }
  for (int d = kWave / 2; d > 0; d >>= 1)
    mine = join_lanes(mine, d, q.c);
  arrived(x_tok);
  const RowCoefs o = finish_row<NT, LOSS>(q, r, mine, x_tok, counted, sh, threadIdx.x == 0);
  if (dx == nullptr) return;
  if (!o.live) {
    zero_gradient<T, NT>(dx, 0, a.vocab);
    return;
  }
  for (int64_t j = threadIdx.x * V; j < a.vocab; j += NT * V) {
    float v[V];
    load(j, v);
#pragma unroll
    for (int e = 0; e < V; ++e) {
      v[e] = gradient_of(v[e], o);
      if (j + e == tok) v[e] += o.at;
    }
    if (j + V <= a.vocab) store_piece(dx + j, v);
    else
      for (int e = 0; e < V; ++e)
        if (j + e < a.vocab) dx[j + e] = static_cast<T>(v[e]);
  }
}

template <class T, bool LOSS>
int launch_rows(const LossKernelArgs& q, RowPart* parts, hipStream_t st) {
  const int64_t rows = q.a.rows, vocab = q.a.vocab, pieces = ceil_div(vocab, kVec<T>), n = ceil_div(pieces, kPartThreads * kPartPieces);
  const dim3 grid = row_grid(rows);
  if (rows <= (LOSS ? kSplitLossRows : kSplitRows) && vocab >= (LOSS ? kSplitLossVocab : kSplitVocab) && n <= kMaxParts) {
    const dim3 split(static_cast<uint32_t>(n), static_cast<uint32_t>(rows));
    hipLaunchKernelGGL(token_part_kernel<T>, split, dim3(kPartThreads), 0, st, q, parts);
    if (int rc = check_launch("token_part_kernel")) return rc;
    if (LOSS) {
      hipLaunchKernelGGL(token_part_gradient_kernel<T>, dim3(split.x, split.y + 1), dim3(kPartThreads), 0, st, q, parts);
      return check_launch("token_part_gradient_kernel");
    }
    hipLaunchKernelGGL(token_joined_kernel, grid, dim3(kWave), 0, st, q, parts, static_cast<int>(n));
    return check_launch("token_joined_kernel");
  }
  // As few threads to a row as hold it, so that a compute unit has several rows in different phases.
#define PPO_ROWS(NT, K) hipLaunchKernelGGL((token_row_kernel<T, NT, K, LOSS>), grid, dim3(NT), 0, st, q)
  if (vocab < kVec<T> || pieces > 1024 * 25)
    hipLaunchKernelGGL((token_wide_kernel<T, LOSS>), grid, dim3(kWideThreads), 0, st, q);
  else if (pieces <= 64) PPO_ROWS(64, 1);
  else if (pieces <= 64 * 4) PPO_ROWS(64, 4);
  else if (pieces <= 256 * 4) PPO_ROWS(256, 4);
  else if (pieces <= 256 * 8) PPO_ROWS(256, 8);
  else if (pieces <= 256 * 16) PPO_ROWS(256, 16);
  else if (pieces <= 512 * 16) PPO_ROWS(512, 16);
  else if (pieces <= 512 * 25) PPO_ROWS(512, 25);
  else if (pieces <= 1024 * 16) PPO_ROWS(1024, 16);
  else PPO_ROWS(1024, 25);
#undef PPO_ROWS
  if (int rc = check_launch("token_row_kernel")) return rc;
  if (!LOSS) return PPO_OK;
  if (rows <= 1024) hipLaunchKernelGGL(token_stats_kernel<256>, dim3(1), dim3(256), 0, st, q);
  else hipLaunchKernelGGL(token_stats_kernel<1024>, dim3(1), dim3(1024), 0, st, q);
  return check_launch("token_stats_kernel");
}

struct Layout {
  size_t terms, parts, bytes;
};

Layout workspace_for(int64_t rows) {
  Layout l;
  l.terms = 256;
  l.parts = l.terms + static_cast<size_t>(rows) * kTermStride * sizeof(float);
  l.bytes = l.parts + (rows <= kSplitRows ? static_cast<size_t>(rows) * kMaxParts * sizeof(RowPart) : 0);
  return l;
}

int check_apart(const char* who, const ppo_token_loss_args& a, bool loss) {
  const int64_t rows = a.rows, size = type_size(a.type);
  const Rows logits{a.logits, rows, a.vocab * size, a.ld_logits * size};
  const Rows d_logits{loss ? a.d_logits : nullptr, rows, a.vocab * size, a.ld_d_logits * size};
  const Rows in[] = {vector_of(a.tokens, rows * (a.token_type == PPO_TOKENS_I64 ? 8 : 4)), vector_of(a.mask, rows),
                     vector_of(loss ? a.old_logp : nullptr, rows * 4), vector_of(loss ? a.ref_logp : nullptr, rows * 4),
                     vector_of(loss ? a.advantages : nullptr, rows * 4)};
  const Rows out[] = {vector_of(a.logp, rows * 4), vector_of(a.entropy, rows * 4), vector_of(loss ? a.stats : nullptr, 32), d_logits};
  PPO_REQUIRE(rows == 0 || d_logits.at == a.logits || !overlap(d_logits, logits), "%s: d_logits overlaps logits and is not in place", who);
  for (int i = 0; i < 4; ++i) {
    PPO_REQUIRE(rows == 0 || i == 3 || !overlap(out[i], logits), "%s: an output overlaps logits", who);
    for (const Rows& x : in) PPO_REQUIRE(rows == 0 || !overlap(out[i], x), "%s: an output overlaps an input", who);
    for (int k = 0; k < i; ++k) PPO_REQUIRE(rows == 0 || !overlap(out[i], out[k]), "%s: outputs overlap", who);
  }
  return PPO_OK;
}

int run(const char* who, const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream,
        bool loss) {
  PPO_REQUIRE(args != nullptr, "%s: null arguments", who);
  const ppo_token_loss_args& a = *args;
  PPO_REQUIRE(a.rows >= 0 && a.rows < INT32_MAX && a.vocab >= 1 && a.vocab < INT32_MAX, "%s: rows=%lld vocab=%lld", who,
              (long long)a.rows, (long long)a.vocab);
  PPO_REQUIRE(type_ok(a.type), "%s: type=%d", who, a.type);
  PPO_REQUIRE(a.token_type == PPO_TOKENS_I64 || a.token_type == PPO_TOKENS_I32, "%s: token_type=%d", who, a.token_type);
  PPO_REQUIRE(a.temperature >= 1e-6 && a.temperature <= 1e6, "%s: temperature=%g", who, a.temperature);
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
    PPO_REQUIRE(a.d_logits != a.logits || a.ld_d_logits == a.ld_logits, "%s: in place needs the same rows", who);
  } else if (a.rows == 0 || (a.logp == nullptr && a.entropy == nullptr)) {
    return PPO_OK;
  }
  const Layout l = workspace_for(a.rows);
  PPO_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= l.bytes,
              "%s: workspace too small or not 16-byte aligned (%zu < %zu)", who, workspace_bytes, l.bytes);
  if (int rc = check_apart(who, a, loss)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  LossKernelArgs q{};
  q.a = a;
  q.stream = a.rows * a.vocab * type_size(a.type) * (loss && a.d_logits != nullptr ? 2 : 1) > kCacheBytes;
  q.inv_n = static_cast<float*>(workspace);
  q.terms = reinterpret_cast<float*>(static_cast<char*>(workspace) + l.terms);
  RowPart* parts = reinterpret_cast<RowPart*>(static_cast<char*>(workspace) + l.parts);
  q.count = !loss || a.denom > 0.0 ? 0 : a.rows <= kCountRows ? 1 : 2;
  q.given_inv_n = a.denom > 0.0 ? static_cast<float>(1.0 / a.denom) : 0.0f;
  q.inv_temp = static_cast<float>(1.0 / a.temperature);
  q.c = static_cast<float>(1.4426950408889634 / a.temperature);
  q.clip_lo = static_cast<float>(1.0 - a.clip_low);
  q.clip_hi = static_cast<float>(1.0 + a.clip_high);
  q.kl_coef = static_cast<float>(a.kl_coef);
  q.entropy_coef = static_cast<float>(a.entropy_coef);
  if (q.count == 2) {
    hipLaunchKernelGGL(token_count_kernel, dim3(1), dim3(kCountThreads), 0, st, q);
    if (int rc = check_launch("token_count_kernel")) return rc;
  }
  if (a.rows > 0) {
    int rc = PPO_OK;
    with_type(a.type, [&](auto t) {
      using T = decltype(t);
      rc = loss ? launch_rows<T, true>(q, parts, st) : launch_rows<T, false>(q, parts, st);
    });
    return rc;
  }
  hipLaunchKernelGGL(token_stats_kernel<256>, dim3(1), dim3(256), 0, st, q);  // no rows: zeros
  return check_launch("token_stats_kernel");
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_token_loss_workspace_bytes(int64_t rows, int64_t vocab) {
  if (rows < 0 || rows >= INT32_MAX || vocab < 1 || vocab >= INT32_MAX) return 0;
  return workspace_for(rows).bytes;
}

extern "C" int ppo_token_log_probs(const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes,
                                   ppo_stream_t stream) {
  return run("ppo_token_log_probs", args, workspace, workspace_bytes, stream, false);
}

extern "C" int ppo_token_ppo_loss(const ppo_token_loss_args* args, void* workspace, size_t workspace_bytes,
                                  ppo_stream_t stream) {
  return run("ppo_token_ppo_loss", args, workspace, workspace_bytes, stream, true);
}
