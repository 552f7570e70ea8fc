// Embedding lookup with scaling, and its gradient by sorted tokens.
//
//   forward    out[i] = s table[tok_i]: rows copied through registers.
//   gradient   dtable[v] = s sum_{i: tok_i = v} dout[i].  The tokens are sorted (stable counting sorts over 9 bits of the token
//              at a time), so that a row's summands lie side by side and are added in the order of i: no atomics on the
//              sums, the same bits on every run, and a frequent token costs no more than as many rare ones.
//
// Both are bound by memory: what they compute is one multiply or add per element.
#include "elem.hpp"

namespace ppo {
namespace {

// ---- forward ----

constexpr int kFwdThreads = 256, kFwdRows = 4;  // rows in flight per thread

template <class T>
__global__ __launch_bounds__(kFwdThreads) void embedding_fwd_kernel(const ppo_embedding_args a, int log_tpr) {
  constexpr int V = kVec<T>;
  const int tpr = 1 << log_tpr;  // threads side by side on a row
  const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x >> log_tpr, groups = kFwdThreads >> log_tpr;
  const int64_t r0 = static_cast<int64_t>(blockIdx.x) * groups * kFwdRows + group;
  const T* table = static_cast<const T*>(a.src);
  T* out = static_cast<T*>(a.dst);
  int64_t tok[kFwdRows];
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    const int64_t i = r0 + u * groups;
    tok[u] = i < a.count ? token_at(a.tokens, a.token_type, i, a.vocab) : -1;
  }
  const int c_step = tpr * V * gridDim.y;
  for (int c0 = (lane + blockIdx.y * tpr) * V; c0 < a.dim; c0 += c_step) {
    if (a.dim >= V) {
      const int c = min(c0, a.dim - V);  // the last piece of an odd row overlaps the one before: the same values twice
      typename Piece<T>::type x[kFwdRows];
#pragma unroll
      for (int u = 0; u < kFwdRows; ++u)
        x[u] = load_piece(table + (tok[u] < 0 ? 0 : tok[u]) * a.ld_src + c);
#pragma unroll
      for (int u = 0; u < kFwdRows; ++u) {
        const int64_t i = r0 + u * groups;
        if (i >= a.count) break;
        float y[V];
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = tok[u] < 0 ? 0.0f : a.scale * static_cast<float>(x[u][e]);
        store_piece(out + i * a.ld_dst + c, y);
      }
    } else {
      for (int u = 0; u < kFwdRows; ++u) {
        const int64_t i = r0 + u * groups;
        if (i >= a.count) break;
        for (int c = c0; c < a.dim; ++c)
          out[i * a.ld_dst + c] =
              static_cast<T>(tok[u] < 0 ? 0.0f : a.scale * static_cast<float>(table[tok[u] * a.ld_src + c]));
      }
    }
  }
}

// ---- the sort ----

constexpr int kTile = 4096, kSortThreads = 1024, kSortWaves = kSortThreads / kWave, kRounds = kTile / kSortThreads;
constexpr int kMaxBits = 9, kMaxDigits = 1 << kMaxBits;

struct SortPlan {
  int passes, bits;  // digits of `bits` bits, `passes` of them
  int tiles;
  int digits() const { return 1 << bits; }
};

SortPlan sort_plan(int64_t count, int64_t vocab) {
  int need = 1;
  while ((int64_t{1} << need) <= vocab) ++need;  // keys 0 .. vocab: what is no token goes to the end as `vocab`
  SortPlan p;
  p.passes = static_cast<int>(ceil_div(need, kMaxBits));
  p.bits = static_cast<int>(ceil_div(need, p.passes));
  p.tiles = static_cast<int>(ceil_div(count, kTile));
  return p;
}

// Items of a tile lie as wave, round, lane: each wave owns kRounds * 64 consecutive ones.
__device__ __forceinline__ int item_in_tile(int round) {
  return (threadIdx.x / kWave) * (kRounds * kWave) + round * kWave + (threadIdx.x & (kWave - 1));
}

__device__ __forceinline__ uint32_t key_at(const ppo_embedding_args& a, int64_t i) {
  const int64_t t = token_at(a.tokens, a.token_type, i, a.vocab);
  return static_cast<uint32_t>(t < 0 ? a.vocab : t);
}

// Stable ranks of a tile's digits: rank[r] counts the items of the same digit before this one in its wave, and
// counts[wave][digit] becomes how many the wave holds.  counts is zero on entry.
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[kRounds], const bool (&in)[kRounds], int bits,
                                           uint32_t* counts, uint32_t (&rank)[kRounds]) {
  uint32_t* mine = counts + (threadIdx.x / kWave) * kMaxDigits;
  const uint64_t below = (uint64_t{1} << (threadIdx.x & (kWave - 1))) - 1;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    uint64_t same = __ballot(in[r]);
    for (int b = 0; b < bits; ++b) {
      const bool set = (digit[r] >> b) & 1;
      const uint64_t m = __ballot(set);
      same &= set ? m : ~m;
    }
    const uint32_t before = __popcll(same & below);
    const uint32_t base = in[r] ? mine[digit[r]] : 0;
    rank[r] = base + before;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read the count before it grows
    if (in[r] && before == 0) mine[digit[r]] = base + __popcll(same);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// counts[wave][digit] -> the items of that digit in earlier waves; returns the tile's number of the thread's digit.
__device__ __forceinline__ uint32_t digit_totals(uint32_t* counts, int digits) {
  uint32_t s = 0;
  if (static_cast<int>(threadIdx.x) < digits)
    for (int w = 0; w < kSortWaves; ++w) {
      const uint32_t c = counts[w * kMaxDigits + threadIdx.x];
      counts[w * kMaxDigits + threadIdx.x] = s;
      s += c;
    }
  return s;
}

// Exclusive sums over the threads' values, for threads below kMaxDigits (the others pass 0).
__device__ __forceinline__ uint32_t exclusive_sum(uint32_t x, uint32_t* scratch /* [kSortWaves] */) {
  uint32_t s = x;
  const int lane = threadIdx.x & (kWave - 1), wave = threadIdx.x / kWave;
  for (int d = 1; d < kWave; d <<= 1) {
    const uint32_t y = __shfl_up(s, d, kWave);
    if (lane >= d) s += y;
  }
  if (lane == kWave - 1) scratch[wave] = s;
  __syncthreads();
  for (int w = 0; w < wave; ++w) s += scratch[w];
  __syncthreads();
  return s - x;
}

__device__ __forceinline__ void clear_counts(uint32_t* counts) {
  for (int i = threadIdx.x; i < kSortWaves * kMaxDigits; i += kSortThreads) counts[i] = 0;
}

// Up to kTile tokens: all passes in one block.
__global__ __launch_bounds__(kSortThreads) void sort_tile_kernel(const ppo_embedding_args a, int passes, int bits,
                                                                 uint32_t* __restrict__ keys, uint32_t* __restrict__ idx) {
  __shared__ uint32_t counts[kSortWaves * kMaxDigits], s_key[kTile], start[kMaxDigits], scratch[kSortWaves];
  __shared__ uint16_t s_idx[kTile];
  const int n = static_cast<int>(a.count);
  uint32_t key[kRounds], from[kRounds], digit[kRounds], rank[kRounds];
  bool in[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int i = item_in_tile(r);
    in[r] = i < n;
    key[r] = in[r] ? key_at(a, i) : 0;
    from[r] = i;
  }
  for (int p = 0; p < passes; ++p) {
    clear_counts(counts);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r) digit[r] = (key[r] >> (p * bits)) & ((1u << bits) - 1);
    wave_ranks(digit, in, bits, counts, rank);
    __syncthreads();
    const uint32_t total = digit_totals(counts, 1 << bits);
    const uint32_t first = exclusive_sum(total, scratch);
    if (threadIdx.x < kMaxDigits) start[threadIdx.x] = first;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (in[r]) {
        const uint32_t to = start[digit[r]] + counts[(threadIdx.x / kWave) * kMaxDigits + digit[r]] + rank[r];
        s_key[to] = key[r];
        s_idx[to] = static_cast<uint16_t>(from[r]);
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < kRounds; ++r)
      if (in[r]) {
        key[r] = s_key[item_in_tile(r)];
        from[r] = s_idx[item_in_tile(r)];
      }
  }
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (in[r]) {
      keys[item_in_tile(r)] = key[r];
      idx[item_in_tile(r)] = from[r];
    }
}

// One pass over several tiles: how many items of each digit a tile holds, hist[digit][tile]; then every item to its place.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const ppo_embedding_args a, int shift, int bits, int tiles,
                                                                  const uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ hist) {
  __shared__ uint32_t count[kMaxDigits];
  if (threadIdx.x < kMaxDigits) count[threadIdx.x] = 0;
  __syncthreads();
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    if (i < a.count) atomicAdd(&count[((keys != nullptr ? keys[i] : key_at(a, i)) >> shift) & ((1u << bits) - 1)], 1u);
  }
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < (1 << bits)) hist[static_cast<int64_t>(threadIdx.x) * tiles + blockIdx.x] = count[threadIdx.x];
}

__global__ __launch_bounds__(kSortThreads) void sort_move_kernel(const ppo_embedding_args a, int shift, int bits, int tiles,
                                                                 const uint32_t* __restrict__ hist,
                                                                 const uint32_t* __restrict__ keys_in,
                                                                 const uint32_t* __restrict__ idx_in,
                                                                 uint32_t* __restrict__ keys, uint32_t* __restrict__ idx) {
  __shared__ uint32_t counts[kSortWaves * kMaxDigits], start[kMaxDigits], scratch[kSortWaves];
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  uint32_t key[kRounds], from[kRounds], digit[kRounds], rank[kRounds];
  bool in[kRounds];
  clear_counts(counts);
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + item_in_tile(r);
    in[r] = i < a.count;
    key[r] = in[r] ? (keys_in != nullptr ? keys_in[i] : key_at(a, i)) : 0;
    from[r] = in[r] ? (idx_in != nullptr ? idx_in[i] : static_cast<uint32_t>(i)) : 0;
    digit[r] = (key[r] >> shift) & ((1u << bits) - 1);
  }
  uint32_t all = 0, earlier = 0;  // items of this thread's digit: in all tiles, in earlier tiles
  if (static_cast<int>(threadIdx.x) < (1 << bits)) {
    const uint32_t* h = hist + static_cast<int64_t>(threadIdx.x) * tiles;
    for (int t = 0; t < tiles; ++t) {
      const uint32_t c = h[t];
      all += c;
      earlier += t < static_cast<int>(blockIdx.x) ? c : 0;
    }
  }
  __syncthreads();
  wave_ranks(digit, in, bits, counts, rank);
  __syncthreads();
  digit_totals(counts, 1 << bits);
  const uint32_t first = exclusive_sum(all, scratch);
  if (threadIdx.x < kMaxDigits) start[threadIdx.x] = first + earlier;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
    if (in[r]) {
      const uint32_t to = start[digit[r]] + counts[(threadIdx.x / kWave) * kMaxDigits + digit[r]] + rank[r];
      keys[to] = key[r];
      idx[to] = from[r];
    }
}

// ---- the sums ----

// The sorted positions are cut into units of kUnit; a wave sums a unit's rows over 64 16-byte pieces of columns.  A run of
// one token inside a unit is stored at once; the parts of a run that crosses units go to `partial` ([units][2][dim]: the
// part of a run that began earlier, and of the one that goes on) and are joined by join_kernel in the units' order.
constexpr int kUnit = 32, kFlight = 8;  // kFlight rows' loads in flight per wave
constexpr int kFillRows = 64;

struct SumArgs {
  ppo_embedding_args e;
  const uint32_t* keys;
  const uint32_t* idx;
  float* partial;
  int64_t ld_partial;
  uint32_t units;
};

template <class T>
__device__ __forceinline__ void store_sum(T* row, int c0, int c, int dim, const float* sum, int n, float scale, bool add) {
  // columns c0 .. of the row; sum[i] is column c + i
  for (int i = 0; i < n; ++i)
    if (c + i >= c0 && c + i < dim)
      row[c + i] = static_cast<T>(add ? static_cast<float>(row[c + i]) + scale * sum[i] : scale * sum[i]);
}

template <class T, class O>
__global__ __launch_bounds__(kWave) void embedding_sum_kernel(const SumArgs s) {
  constexpr int V = kVec<T>;
  const ppo_embedding_args& a = s.e;
  const int lane = threadIdx.x;
  const uint32_t n = static_cast<uint32_t>(a.count);
  O* out = static_cast<O*>(a.dst);
  if (blockIdx.x >= s.units) {  // rows without tokens become zero
    const int64_t v0 = static_cast<int64_t>(blockIdx.x - s.units) * kFillRows, v = v0 + lane;
    uint32_t lo = 0, hi = n;
    while (lo < hi) {
      const uint32_t mid = (lo + hi) / 2;
      if (s.keys[mid] < v) lo = mid + 1;
      else hi = mid;
    }
    uint64_t empty = __ballot(v < a.vocab && (lo >= n || s.keys[lo] != v));
    while (empty != 0) {
      const int r = __ffsll(static_cast<unsigned long long>(empty)) - 1;
      empty &= empty - 1;
      O* row = out + (v0 + r) * a.ld_dst;
      constexpr int W = kVec<O>;
      const float zero[W] = {};
      for (int c = (lane + blockIdx.y * kWave) * W; c < a.dim; c += kWave * W * gridDim.y) {
        if (c + W <= a.dim) store_piece(row + c, zero);
        else
          for (int i = c; i < a.dim; ++i) row[i] = static_cast<O>(0.0f);
      }
    }
    return;
  }
  const int c0 = (blockIdx.y * kWave + lane) * V;
  if (c0 >= a.dim) return;
  const bool whole = a.dim >= V;
  const int c = whole ? min(c0, a.dim - V) : 0;  // an odd row's last piece is read from V columns before its end
  const T* src = static_cast<const T*>(a.src);
  const uint32_t begin = blockIdx.x * kUnit, end = min(begin + kUnit, n);
  uint32_t cur = s.keys[begin];
  bool head = begin > 0 && s.keys[begin - 1] == cur;  // the run began in an earlier unit
  float sum[V] = {};
  auto flush = [&](bool tail) {
    if (cur < a.vocab) {
      if (head || tail) {
        float* to = s.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (head ? 0 : 1)) * s.ld_partial;
        for (int i = 0; i < V; ++i)
          if (c + i >= c0 && c + i < a.dim) to[c + i] = sum[i];
      } else {
        store_sum(out + static_cast<int64_t>(cur) * a.ld_dst, c0, c, a.dim, sum, V, a.scale, a.accumulate != 0);
      }
    }
    head = false;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  };
  for (uint32_t p = begin; p < end; p += kFlight) {
    typename Piece<T>::type x[kFlight];
    uint32_t key[kFlight];
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const uint32_t q = min(p + u, end - 1);
      key[u] = s.keys[q];
      const T* row = src + static_cast<int64_t>(s.idx[q]) * a.ld_src;
      if (whole) {
        x[u] = load_piece(row + c);
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) x[u][i] = i < a.dim ? row[i] : static_cast<T>(0.0f);
      }
    }
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (p + u >= end) break;
      if (key[u] != cur) {
        flush(false);
        cur = key[u];
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += static_cast<float>(x[u][i]);
    }
  }
  flush(end < n && s.keys[end] == cur);
}

// A run that crosses units: the unit where it begins adds the parts of the units it goes on in.
constexpr int kJoinThreads = 256;

template <class O>
__global__ __launch_bounds__(kJoinThreads) void embedding_join_kernel(const SumArgs s) {
  const ppo_embedding_args& a = s.e;
  const uint32_t n = static_cast<uint32_t>(a.count), u = blockIdx.x;
  const uint32_t begin = u * kUnit, end = min(begin + kUnit, n);
  if (end >= n) return;
  const uint32_t key = s.keys[end - 1];
  if (s.keys[end] != key || key >= a.vocab) return;             // the last run ends with the unit
  if (s.keys[begin] == key && begin > 0 && s.keys[begin - 1] == key) return;  // it began in an earlier one
  const int c = blockIdx.y * kJoinThreads + threadIdx.x;
  if (c >= a.dim) return;
  float sum = s.partial[(static_cast<int64_t>(u) * 2 + 1) * s.ld_partial + c];
  for (uint32_t w = u + 1; w < s.units && s.keys[w * kUnit] == key; ++w)
    sum += s.partial[static_cast<int64_t>(w) * 2 * s.ld_partial + c];
  O* to = static_cast<O*>(a.dst) + static_cast<int64_t>(key) * a.ld_dst + c;
  *to = static_cast<O>(a.accumulate ? static_cast<float>(*to) + a.scale * sum : a.scale * sum);
}

int check(const char* who, const ppo_embedding_args* a, bool bwd) {
  PPO_REQUIRE(a != nullptr, "%s: null arguments", who);
  PPO_REQUIRE(a->count >= 0 && a->count < INT32_MAX && a->vocab >= 1 && a->vocab < INT32_MAX && a->dim >= 1,
              "%s: count=%lld vocab=%lld dim=%d", who, (long long)a->count, (long long)a->vocab, a->dim);
  PPO_REQUIRE(type_ok(a->src_type) && type_ok(a->dst_type), "%s: src_type=%d dst_type=%d", who, a->src_type, a->dst_type);
  PPO_REQUIRE(a->dst_type == a->src_type || (bwd && a->dst_type == PPO_TYPE_F32),
              "%s: dst_type=%d for src_type=%d", who, a->dst_type, a->src_type);
  PPO_REQUIRE(a->token_type == PPO_TOKENS_I64 || a->token_type == PPO_TOKENS_I32, "%s: token_type=%d", who, a->token_type);
  PPO_REQUIRE(a->ld_src >= a->dim && a->ld_dst >= a->dim, "%s: leading dimensions %lld, %lld below dim=%d", who,
              (long long)a->ld_src, (long long)a->ld_dst, a->dim);
  PPO_REQUIRE(a->dst != nullptr || (!bwd && a->count == 0), "%s: null pointer", who);
  PPO_REQUIRE(a->count == 0 || (a->tokens != nullptr && a->src != nullptr), "%s: null pointer", who);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a->src) % type_size(a->src_type) == 0 &&
                  reinterpret_cast<uintptr_t>(a->dst) % type_size(a->dst_type) == 0 &&
                  reinterpret_cast<uintptr_t>(a->tokens) % (a->token_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  return PPO_OK;
}

struct BwdLayout {
  SortPlan sort;
  uint32_t units;
  int64_t ld_partial;
  size_t keys[2], idx[2], hist, partial, bytes;
};

BwdLayout bwd_layout(int64_t count, int64_t vocab, int32_t dim) {
  BwdLayout l{};
  l.sort = sort_plan(count, vocab);
  l.units = static_cast<uint32_t>(ceil_div(count, kUnit));
  l.ld_partial = ceil_div(dim, 4) * 4;
  size_t at = 0;
  auto take = [&](size_t bytes) {
    const size_t here = at;
    at += (bytes + 255) / 256 * 256;
    return here;
  };
  for (int k = 0; k < 2; ++k) {
    l.keys[k] = take(4 * static_cast<size_t>(count));
    l.idx[k] = take(4 * static_cast<size_t>(count));
  }
  l.hist = take(l.sort.tiles > 1 ? 4 * static_cast<size_t>(l.sort.digits()) * l.sort.tiles : 0);
  l.partial = take(8 * static_cast<size_t>(l.units) * l.ld_partial);
  l.bytes = at;
  return l;
}

template <class T, class O>
int launch_sums(const SumArgs& s, int64_t fill, hipStream_t st) {
  const int dim = s.e.dim;
  const dim3 grid(static_cast<uint32_t>(s.units + fill), static_cast<uint32_t>(ceil_div(dim, kWave * kVec<T>)));
  hipLaunchKernelGGL((embedding_sum_kernel<T, O>), grid, dim3(kWave), 0, st, s);
  if (int rc = check_launch("embedding_sum_kernel")) return rc;
  if (s.units < 2) return PPO_OK;
  const dim3 join(s.units - 1, static_cast<uint32_t>(ceil_div(dim, kJoinThreads)));
  hipLaunchKernelGGL(embedding_join_kernel<O>, join, dim3(kJoinThreads), 0, st, s);
  return check_launch("embedding_join_kernel");
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" int ppo_embedding_fwd(const ppo_embedding_args* args, ppo_stream_t stream) {
  if (int rc = check("ppo_embedding_fwd", args, false)) return rc;
  const ppo_embedding_args& a = *args;
  if (a.count == 0) return PPO_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = PPO_OK;
  with_type(a.src_type, [&](auto t) {
    using T = decltype(t);
    const int64_t pieces = ceil_div(a.dim, kVec<T>);
    int log_tpr = 0;
    while ((1 << log_tpr) < pieces && (1 << log_tpr) < kFwdThreads) ++log_tpr;
    const int64_t blocks = ceil_div(a.count, static_cast<int64_t>(kFwdThreads >> log_tpr) * kFwdRows);
    hipLaunchKernelGGL(embedding_fwd_kernel<T>, dim3(static_cast<uint32_t>(blocks)), dim3(kFwdThreads), 0, st, a, log_tpr);
    rc = check_launch("embedding_fwd_kernel");
  });
  return rc;
}

extern "C" size_t ppo_embedding_bwd_workspace_bytes(int64_t count, int64_t vocab, int32_t dim) {
  if (count < 0 || count >= INT32_MAX || vocab < 1 || vocab >= INT32_MAX || dim < 1) return 0;
  return bwd_layout(count, vocab, dim).bytes;
}

extern "C" int ppo_embedding_bwd(const ppo_embedding_args* args, void* workspace, size_t workspace_bytes,
                                 ppo_stream_t stream) {
  if (int rc = check("ppo_embedding_bwd", args, true)) return rc;
  const ppo_embedding_args& a = *args;
  const BwdLayout l = bwd_layout(a.count, a.vocab, a.dim);
  PPO_REQUIRE(workspace_bytes >= l.bytes && (workspace != nullptr || l.bytes == 0),
              "ppo_embedding_bwd: workspace too small (%zu < %zu)", workspace_bytes, l.bytes);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "ppo_embedding_bwd: the workspace must be 16-byte aligned");
  if (a.count == 0 && a.accumulate) return PPO_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  auto at = [&](size_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
  int last = 0;  // the buffer that holds the sorted tokens
  if (l.sort.tiles == 1) {
    hipLaunchKernelGGL(sort_tile_kernel, dim3(1), dim3(kSortThreads), 0, st, a, l.sort.passes, l.sort.bits, at(l.keys[0]),
                       at(l.idx[0]));
    if (int rc = check_launch("sort_tile_kernel")) return rc;
  } else if (l.sort.tiles > 1) {
    for (int p = 0; p < l.sort.passes; ++p) {
      const int to = p & 1, from = 1 - to, shift = p * l.sort.bits;
      const uint32_t* keys = p == 0 ? nullptr : at(l.keys[from]);
      const uint32_t* idx = p == 0 ? nullptr : at(l.idx[from]);
      hipLaunchKernelGGL(sort_count_kernel, dim3(l.sort.tiles), dim3(kSortThreads), 0, st, a, shift, l.sort.bits, l.sort.tiles,
                         keys, at(l.hist));
      if (int rc = check_launch("sort_count_kernel")) return rc;
      hipLaunchKernelGGL(sort_move_kernel, dim3(l.sort.tiles), dim3(kSortThreads), 0, st, a, shift, l.sort.bits, l.sort.tiles,
                         at(l.hist), keys, idx, at(l.keys[to]), at(l.idx[to]));
      if (int rc = check_launch("sort_move_kernel")) return rc;
      last = to;
    }
  }
  SumArgs s{a, at(l.keys[last]), at(l.idx[last]), reinterpret_cast<float*>(ws + l.partial), l.ld_partial, l.units};
  const int64_t fill = a.accumulate ? 0 : ceil_div(a.vocab, kFillRows);
  int rc = PPO_OK;
  with_type(a.src_type, [&](auto t) {
    using T = decltype(t);
    if (a.dst_type == PPO_TYPE_F32) rc = launch_sums<T, float>(s, fill, st);
    else rc = launch_sums<T, T>(s, fill, st);
  });
  return rc;
}
