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

// Items of a tile lie as wave, round, lane: each wave owns ROUNDS * 64 consecutive ones.  Up to kOneTile tokens are sorted
// by one block in one launch; more go in tiles of kTile, two launches for each 9 bits of the token.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kTileRounds = 4, kTile = kTileRounds * kSortThreads, kOneRounds = 8, kOneTile = kOneRounds * kSortThreads;
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
  p.tiles = count == 0 ? 0 : count <= kOneTile ? 1 : static_cast<int>(ceil_div(count, kTile));
  return p;
}

// The gradient's rows become zero by blocks of the sort's launches, which leave most of the chip idle; rows with tokens are
// written again by the sums.  Block b of a launch fills bytes [b kFillBytes, (b + 1) kFillBytes) of a gapless table, or as
// many whole rows, from `first` on.
constexpr int64_t kFillBytes = 1 << 17;

struct Fill {
  char* dst;
  int64_t rows, row_bytes, ld_bytes;
  int64_t first;  // blocks of earlier launches
};

__device__ __forceinline__ void store_zeros(char* p, int64_t bytes, int lane, int lanes) {
  // from an address of the element's alignment on; the ends by 2 bytes
  const int64_t head = min<int64_t>(bytes, -reinterpret_cast<intptr_t>(p) & 15);
  const int64_t pieces = (bytes - head) / 16, tail = head + pieces * 16;
  for (int64_t i = lane; i < pieces; i += lanes) *reinterpret_cast<float4*>(p + head + 16 * i) = float4{0.0f, 0.0f, 0.0f, 0.0f};
  for (int64_t i = 2 * lane; i < head; i += 2 * lanes) *reinterpret_cast<uint16_t*>(p + i) = 0;
  for (int64_t i = tail + 2 * lane; i < bytes; i += 2 * lanes) *reinterpret_cast<uint16_t*>(p + i) = 0;
}

__device__ __forceinline__ void fill_block(const Fill& f, int64_t block) {
  block += f.first;
  if (f.ld_bytes == f.row_bytes) {
    const int64_t from = block * kFillBytes;
    store_zeros(f.dst + from, min<int64_t>(kFillBytes, f.rows * f.row_bytes - from), threadIdx.x, kSortThreads);
    return;
  }
  const int64_t per = max<int64_t>(1, kFillBytes / f.row_bytes), end = min<int64_t>(f.rows, (block + 1) * per);
  for (int64_t r = block * per + threadIdx.x / kWave; r < end; r += kSortWaves)  // a wave per row
    store_zeros(f.dst + r * f.ld_bytes, f.row_bytes, threadIdx.x % kWave, kWave);
}

int64_t fill_blocks(const Fill& f) {
  return f.ld_bytes == f.row_bytes ? ceil_div(f.rows * f.row_bytes, kFillBytes)
                                   : ceil_div(f.rows, std::max<int64_t>(1, kFillBytes / f.row_bytes));
}

__device__ __forceinline__ uint32_t key_at(const ppo_embedding_args& a, int64_t i) {
  const int64_t t = token_at(a.tokens, a.token_type, i, a.vocab);
  return static_cast<uint32_t>(t < 0 ? a.vocab : t);
}

template <int ROUNDS>
__device__ __forceinline__ int item_in_tile(int round) {
  return (threadIdx.x / kWave) * (ROUNDS * kWave) + round * kWave + (threadIdx.x & (kWave - 1));
}

// Stable ranks of a tile's digits: rank[r] counts the items of the same digit before this one in its wave, and
// counts[wave][digit] becomes how many the wave holds.  counts is zero on entry.  The lanes of a digit find each other by a
// ballot per bit.
template <int ROUNDS>
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[ROUNDS], const bool (&in)[ROUNDS], int bits,
                                           uint32_t* counts, uint32_t (&rank)[ROUNDS]) {
  uint32_t* mine = counts + (threadIdx.x / kWave) * kMaxDigits;
  const uint64_t below = (uint64_t{1} << (threadIdx.x & (kWave - 1))) - 1;
  uint64_t same[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) same[r] = __ballot(in[r]);
#pragma unroll
  for (int b = 0; b < kMaxBits; ++b)
    if (b < bits) {
#pragma unroll
      for (int r = 0; r < ROUNDS; ++r) {
        const bool set = (digit[r] >> b) & 1;
        const uint64_t m = __ballot(set);
        same[r] &= set ? m : ~m;
      }
    }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const uint32_t before = __popcll(same[r] & below);
    const uint32_t base = in[r] ? mine[digit[r]] : 0;
    rank[r] = base + before;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");  // every lane has read the count before it grows
    if (in[r] && before == 0) mine[digit[r]] = base + __popcll(same[r]);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
  }
}

// counts[wave][digit] -> the items of that digit in earlier waves; returns the tile's number of the thread's digit.
__device__ __forceinline__ uint32_t digit_totals(uint32_t* counts, int digits) {
  uint32_t s = 0;
  if (static_cast<int>(threadIdx.x) < digits) {
    uint32_t c[kSortWaves];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) c[w] = counts[w * kMaxDigits + threadIdx.x];
#pragma unroll
    for (int w = 0; w < kSortWaves; ++w) {
      counts[w * kMaxDigits + threadIdx.x] = s;
      s += c[w];
    }
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
  uint32_t before = 0;
#pragma unroll
  for (int w = 0; w < kMaxDigits / kWave; ++w) before += w < wave ? scratch[w] : 0;
  __syncthreads();
  return s + before - x;
}

__device__ __forceinline__ void clear_counts(uint32_t* counts) {
#pragma unroll
  for (int i = 0; i < kSortWaves * kMaxDigits / kSortThreads; ++i) counts[i * kSortThreads + threadIdx.x] = 0;
}

// Up to kOneTile tokens: all passes in one block.
__global__ __launch_bounds__(kSortThreads) void sort_tile_kernel(const ppo_embedding_args a, int passes, int bits,
                                                                 uint32_t* __restrict__ keys, uint32_t* __restrict__ idx,
                                                                 const Fill fill) {
  constexpr int ROUNDS = kOneRounds;
  __shared__ uint32_t counts[kSortWaves * kMaxDigits], s_key[kOneTile], start[kMaxDigits], scratch[kSortWaves];
  __shared__ uint16_t s_idx[kOneTile];
  static_assert(kOneTile <= 1 << 16, "16-bit indices");
  if (blockIdx.x > 0) {
    fill_block(fill, blockIdx.x - 1);
    return;
  }
  const int n = static_cast<int>(a.count);
  uint32_t key[ROUNDS], from[ROUNDS], digit[ROUNDS], rank[ROUNDS];
  bool in[ROUNDS];
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r) {
    const int i = item_in_tile<ROUNDS>(r);
    in[r] = i < n;
    key[r] = in[r] ? key_at(a, i) : 0;
    from[r] = i;
  }
  for (int p = 0; p < passes; ++p) {
    clear_counts(counts);
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r) digit[r] = (key[r] >> (p * bits)) & ((1u << bits) - 1);
    wave_ranks(digit, in, bits, counts, rank);
    __syncthreads();
    const uint32_t total = digit_totals(counts, 1 << bits);
    const uint32_t first = exclusive_sum(total, scratch);
    if (threadIdx.x < kMaxDigits) start[threadIdx.x] = first;
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      if (in[r]) {
        const uint32_t to = start[digit[r]] + counts[(threadIdx.x / kWave) * kMaxDigits + digit[r]] + rank[r];
        s_key[to] = key[r];
        s_idx[to] = static_cast<uint16_t>(from[r]);
      }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < ROUNDS; ++r)
      if (in[r]) {
        key[r] = s_key[item_in_tile<ROUNDS>(r)];
        from[r] = s_idx[item_in_tile<ROUNDS>(r)];
      }
  }
#pragma unroll
  for (int r = 0; r < ROUNDS; ++r)
    if (in[r]) {
      keys[item_in_tile<ROUNDS>(r)] = key[r];
      idx[item_in_tile<ROUNDS>(r)] = from[r];
    }
}

// One pass over several tiles: how many items of each digit a tile holds, hist[tile][digit]; then every item to its place.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const ppo_embedding_args a, int shift, int bits, int tiles,
                                                                  const uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ hist, const Fill fill) {
  __shared__ uint32_t count[kMaxDigits];
  if (static_cast<int>(blockIdx.x) >= tiles) {
    fill_block(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  uint32_t key[kTileRounds];
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    key[r] = i < a.count ? (keys != nullptr ? keys[i] : key_at(a, i)) : 0;
  }
  if (threadIdx.x < kMaxDigits) count[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r)
    if (base + r * kSortThreads + threadIdx.x < a.count) atomicAdd(&count[(key[r] >> shift) & ((1u << bits) - 1)], 1u);
  __syncthreads();
  if (static_cast<int>(threadIdx.x) < (1 << bits)) hist[(static_cast<int64_t>(blockIdx.x) << bits) + threadIdx.x] = count[threadIdx.x];
}

__global__ __launch_bounds__(kSortThreads) void sort_move_kernel(const ppo_embedding_args a, int shift, int bits, int tiles,
                                                                 const uint32_t* __restrict__ hist,
                                                                 const uint32_t* __restrict__ keys_in,
                                                                 const uint32_t* __restrict__ idx_in,
                                                                 uint32_t* __restrict__ keys, uint32_t* __restrict__ idx,
                                                                 const Fill fill) {
  __shared__ uint32_t counts[kSortWaves * kMaxDigits], start[kMaxDigits], scratch[kSortWaves];
  if (static_cast<int>(blockIdx.x) >= tiles) {
    fill_block(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  uint32_t key[kTileRounds], from[kTileRounds], digit[kTileRounds], rank[kTileRounds];
  bool in[kTileRounds];
  clear_counts(counts);
#pragma unroll
  for (int r = 0; r < kTileRounds; ++r) {
    const int64_t i = base + item_in_tile<kTileRounds>(r);
    in[r] = i < a.count;
    key[r] = in[r] ? (keys_in != nullptr ? keys_in[i] : key_at(a, i)) : 0;
    from[r] = in[r] ? (idx_in != nullptr ? idx_in[i] : static_cast<uint32_t>(i)) : 0;
    digit[r] = (key[r] >> shift) & ((1u << bits) - 1);
  }
  uint32_t all = 0, earlier = 0;  // items of this thread's digit: in all tiles, in earlier tiles
  if (static_cast<int>(threadIdx.x) < (1 << bits)) {
    const uint32_t* h = hist + threadIdx.x;
#pragma unroll 16
    for (int t = 0; t < tiles; ++t) {
      const uint32_t c = h[static_cast<int64_t>(t) << bits];
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
  for (int r = 0; r < kTileRounds; ++r)
    if (in[r]) {
      const uint32_t to = start[digit[r]] + counts[(threadIdx.x / kWave) * kMaxDigits + digit[r]] + rank[r];
      keys[to] = key[r];
      idx[to] = from[r];
    }
}

__global__ __launch_bounds__(kSortThreads) void fill_kernel(const Fill fill) { fill_block(fill, blockIdx.x); }

// ---- the sums ----

// The sorted positions are cut into units; a wave sums a unit's rows over 64 16-byte pieces of columns.  A run of
// one token inside a unit is stored at once; the parts of a run that crosses units go to `partial` ([units][2][dim]: the
// part of a run that began earlier, and of the one that goes on) and are joined by join_kernel in the units' order.
constexpr int kFlight = 8;  // rows' loads in flight per wave

struct SumArgs {
  ppo_embedding_args e;
  const uint32_t* keys;
  const uint32_t* idx;
  float* partial;
  int64_t ld_partial;  // a multiple of 4
  uint32_t unit;       // positions
  uint32_t units;
};

// sum[i] is column c + i of the row; columns from c0 on are this lane's.
template <int V, class T>
__device__ __forceinline__ void store_sum(T* row, int c0, int c, int dim, const float (&sum)[V], float scale, bool add) {
  constexpr int W = kVec<T> < V ? kVec<T> : V;  // (fp32 rows from 16-bit summands: two pieces)
  if (c == c0 && dim >= V) {
#pragma unroll
    for (int p = 0; p < V / W; ++p) {
      typedef T vec __attribute__((ext_vector_type(W), aligned(sizeof(T))));
      vec* to = reinterpret_cast<vec*>(row + c + p * W);
      vec v;
      if (add) v = *to;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        const float y = scale * sum[p * W + i];
        v[i] = static_cast<T>(add ? static_cast<float>(v[i]) + y : y);
      }
      *to = v;
    }
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (c + i >= c0 && c + i < dim)
        row[c + i] = static_cast<T>(add ? static_cast<float>(row[c + i]) + scale * sum[i] : scale * sum[i]);
  }
}

template <class T, class O>
__global__ __launch_bounds__(kWave) void embedding_sum_kernel(const SumArgs s) {
  constexpr int V = kVec<T>;
  const ppo_embedding_args& a = s.e;
  const int lane = threadIdx.x;
  const uint32_t n = static_cast<uint32_t>(a.count);
  O* out = static_cast<O*>(a.dst);
  const int c0 = (blockIdx.y * kWave + lane) * V;
  if (c0 >= a.dim) return;
  const bool whole = a.dim >= V;
  const int c = whole ? min(c0, a.dim - V) : 0;  // an odd row's last piece is read from V columns before its end
  const T* src = static_cast<const T*>(a.src);
  const uint32_t begin = blockIdx.x * s.unit, end = min(begin + s.unit, n);
  uint32_t cur = s.keys[begin];
  bool head = begin > 0 && s.keys[begin - 1] == cur;  // the run began in an earlier unit
  float sum[V] = {};
  auto flush = [&](bool tail) {
    if (cur < a.vocab) {
      if (head || tail)
        store_sum<V>(s.partial + (static_cast<int64_t>(blockIdx.x) * 2 + (head ? 0 : 1)) * s.ld_partial, c0, c, a.dim, sum, 1.0f, false);
      else
        store_sum<V>(out + static_cast<int64_t>(cur) * a.ld_dst, c0, c, a.dim, sum, a.scale, a.accumulate != 0);
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

// A run that crosses units: the block of the unit where it begins adds the parts of the units it goes on in, each wave a
// consecutive share of them, and the waves' sums in order.
constexpr int kJoinThreads = 256, kJoinWaves = kJoinThreads / kWave, kJoinColumns = 4 * kWave;

template <class O>
__global__ __launch_bounds__(kJoinThreads) void embedding_join_kernel(const SumArgs s) {
  __shared__ float4 part[kJoinWaves][kWave];
  const ppo_embedding_args& a = s.e;
  const uint32_t n = static_cast<uint32_t>(a.count), u = blockIdx.x;
  const uint32_t begin = u * s.unit, end = min(begin + s.unit, n);
  if (end >= n) return;
  const uint32_t key = s.keys[end - 1];
  if (s.keys[end] != key || key >= a.vocab) return;                           // the last run ends with the unit
  if (s.keys[begin] == key && begin > 0 && s.keys[begin - 1] == key) return;  // it began in an earlier one
  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  uint32_t more = 0;  // units after this one that begin with the same token
  while (true) {
    const uint32_t w = u + 1 + more + lane;
    const uint64_t m = __ballot(w < s.units && s.keys[static_cast<int64_t>(min(w, s.units - 1)) * s.unit] == key);
    more += m == ~uint64_t{0} ? kWave : __ffsll(static_cast<unsigned long long>(~m)) - 1;
    if (m != ~uint64_t{0}) break;
  }
  const int c = (blockIdx.y * kWave + lane) * 4;
  float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
  if (c < a.dim) {
    auto add = [&](const float4& x) { sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w; };
    if (wave == 0) add(*reinterpret_cast<const float4*>(s.partial + (static_cast<int64_t>(u) * 2 + 1) * s.ld_partial + c));
    const uint32_t share = (more + kJoinWaves - 1) / kJoinWaves, last = min(more, (wave + 1) * share);
#pragma unroll 8
    for (uint32_t i = wave * share; i < last; ++i)
      add(*reinterpret_cast<const float4*>(s.partial + static_cast<int64_t>(u + 1 + i) * 2 * s.ld_partial + c));
  }
  part[wave][lane] = sum;
  __syncthreads();
  if (wave > 0 || c >= a.dim) return;
  float x[4] = {};
#pragma unroll
  for (int w = 0; w < kJoinWaves; ++w) {
    const float4 y = part[w][lane];
    x[0] += y.x, x[1] += y.y, x[2] += y.z, x[3] += y.w;
  }
  O* to = static_cast<O*>(a.dst) + static_cast<int64_t>(key) * a.ld_dst + c;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    if (c + i < a.dim) to[i] = static_cast<O>(a.accumulate ? static_cast<float>(to[i]) + a.scale * x[i] : a.scale * x[i]);
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
  uint32_t unit, units;
  int64_t ld_partial;
  size_t keys[2], idx[2], hist, partial, bytes;
};

// Positions of a unit: enough waves to fill the chip (8,192 hold 64 KiB of loads in flight each four SIMDs), but at least 8 rows,
// since a run that crosses units costs a row of partial sums for each, and at most 64.
uint32_t unit_for(int64_t count, int32_t dim) {
  uint32_t unit = 8;
  while (unit < 64 && count * ceil_div(dim, 512) > static_cast<int64_t>(unit) * 8192) unit *= 2;
  return unit;
}

BwdLayout bwd_layout(int64_t count, int64_t vocab, int32_t dim) {
  BwdLayout l{};
  l.sort = sort_plan(count, vocab);
  l.unit = unit_for(count, dim);
  l.units = static_cast<uint32_t>(ceil_div(count, l.unit));
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
int launch_sums(const SumArgs& s, hipStream_t st) {
  const int dim = s.e.dim;
  const dim3 grid(s.units, static_cast<uint32_t>(ceil_div(dim, kWave * kVec<T>)));
  hipLaunchKernelGGL((embedding_sum_kernel<T, O>), grid, dim3(kWave), 0, st, s);
  if (int rc = check_launch("embedding_sum_kernel")) return rc;
  if (s.units < 2) return PPO_OK;
  const dim3 join(s.units - 1, static_cast<uint32_t>(ceil_div(dim, kJoinColumns)));
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
  const int64_t size = type_size(a.dst_type);
  Fill fill{static_cast<char*>(a.dst), a.vocab, a.dim * size, a.ld_dst * size, 0};
  const int64_t blocks = a.accumulate ? 0 : fill_blocks(fill);
  PPO_REQUIRE(blocks < (int64_t{1} << 30), "ppo_embedding_bwd: the table is too large");
  int last = 0;  // the buffer that holds the sorted tokens
  if (l.sort.tiles == 0) {
    hipLaunchKernelGGL(fill_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kSortThreads), 0, st, fill);
    return check_launch("fill_kernel");
  }
  if (l.sort.tiles == 1) {
    hipLaunchKernelGGL(sort_tile_kernel, dim3(1 + static_cast<uint32_t>(blocks)), dim3(kSortThreads), 0, st, a, l.sort.passes,
                       l.sort.bits, at(l.keys[0]), at(l.idx[0]), fill);
    if (int rc = check_launch("sort_tile_kernel")) return rc;
  } else {
    // the launches' shares of the filling, about as their own work lasts: 1 for a count, 2 for a move
    const int64_t share = ceil_div(blocks, 3 * l.sort.passes);
    auto part = [&](int64_t wanted) { return static_cast<uint32_t>(std::min(wanted, blocks - fill.first)); };
    for (int p = 0; p < l.sort.passes; ++p) {
      const int to = p & 1, from = 1 - to, shift = p * l.sort.bits;
      const uint32_t* keys = p == 0 ? nullptr : at(l.keys[from]);
      const uint32_t* idx = p == 0 ? nullptr : at(l.idx[from]);
      uint32_t more = part(share);
      hipLaunchKernelGGL(sort_count_kernel, dim3(l.sort.tiles + more), dim3(kSortThreads), 0, st, a, shift, l.sort.bits,
                         l.sort.tiles, keys, at(l.hist), fill);
      if (int rc = check_launch("sort_count_kernel")) return rc;
      fill.first += more;
      more = part(2 * share);
      hipLaunchKernelGGL(sort_move_kernel, dim3(l.sort.tiles + more), dim3(kSortThreads), 0, st, a, shift, l.sort.bits,
                         l.sort.tiles, at(l.hist), keys, idx, at(l.keys[to]), at(l.idx[to]), fill);
      if (int rc = check_launch("sort_move_kernel")) return rc;
      fill.first += more;
      last = to;
    }
  }
  const SumArgs s{a, at(l.keys[last]), at(l.idx[last]), reinterpret_cast<float*>(ws + l.partial), l.ld_partial, l.unit, l.units};
  int rc = PPO_OK;
  with_type(a.src_type, [&](auto t) {
    using T = decltype(t);
    if (a.dst_type == PPO_TYPE_F32) rc = launch_sums<T, float>(s, st);
    else rc = launch_sums<T, T>(s, st);
  });
  return rc;
}
