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

// A thread moves one 16-byte piece of each of kFwdRows rows; a block's threads lie side by side on a row as far as it reaches.
// 16,384 rows of 2,048 bf16: 17.8 us, 5.2 TB/s of the 93 MB that have to move.
constexpr int kFwdThreads = 256, kFwdRows = 4;  // rows in flight per thread
constexpr int64_t kFwdGrid = 1 << 20;  // blocks along x; more go along z (2^32 threads along one axis are refused)

template <class T>
__global__ __launch_bounds__(kFwdThreads) void embedding_fwd_kernel(const ppo_embedding_args a, int log_tpr) {
  constexpr int V = kVec<T>;
  const int tpr = 1 << log_tpr;  // threads side by side on a row
  const int lane = threadIdx.x & (tpr - 1), group = threadIdx.x >> log_tpr, groups = kFwdThreads >> log_tpr;
  const int64_t r0 = (blockIdx.x + blockIdx.z * kFwdGrid) * groups * kFwdRows + group;
  if (r0 >= a.count) return;
  const T* table = static_cast<const T*>(a.src);
  T* out = static_cast<T*>(a.dst);
  int64_t tok[kFwdRows];
#pragma unroll
  for (int u = 0; u < kFwdRows; ++u) {
    const int64_t i = r0 + u * groups;
    tok[u] = i < a.count ? token_at(a.tokens, a.token_type, i, a.vocab) : -1;
  }
  const int c0 = (lane + blockIdx.y * tpr) * V;
  if (c0 >= a.dim) return;
  if (a.dim >= V) {
    const int c = min(c0, a.dim - V);  // the last piece of an odd row overlaps the one before: the same values twice
    typename Piece<T>::type x[kFwdRows];
#pragma unroll
    for (int u = 0; u < kFwdRows; ++u) x[u] = load_piece(table + (tok[u] < 0 ? 0 : tok[u]) * a.ld_src + c);
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
      for (int c = 0; c < a.dim; ++c)
        out[i * a.ld_dst + c] =
            static_cast<T>(tok[u] < 0 ? 0.0f : a.scale * static_cast<float>(table[tok[u] * a.ld_src + c]));
    }
  }
}

// ---- the sort ----

// Up to kRankMax tokens find their places by comparing each with all (rank_kernel, one launch); more are sorted in tiles of
// kTile, two launches for each 9 bits of the token.  A tile's items lie as wave, round, lane: each wave owns kRounds * 64
// consecutive ones.  Every block of a move reads all tiles' counts, so the sort's work has a part that grows with the square of
// the tokens: 2 MB a pass for 131,072 of them, 34 GB for 16 M.
constexpr int kSortThreads = 1024, kSortWaves = kSortThreads / kWave;
constexpr int kRounds = 4, kTile = kRounds * kSortThreads;
constexpr int64_t kRankMax = 12288;  // (gradients of 12,000 tokens 34 us so, 39 by the other; of 16,384 45 and 39)
constexpr int kMaxBits = 9, kMaxDigits = 1 << kMaxBits;

struct SortPlan {
  int passes, bits;  // digits of `bits` bits, `passes` of them
  int tiles;         // 0: by rank_kernel
  int digits() const { return 1 << bits; }
};

SortPlan sort_plan(int64_t count, int64_t vocab) {
  int need = 1;
  while ((int64_t{1} << need) <= vocab) ++need;  // keys 0 .. vocab: what is no token goes to the end as `vocab`
  SortPlan p;
  p.passes = static_cast<int>(ceil_div(need, kMaxBits));
  p.bits = static_cast<int>(ceil_div(need, p.passes));
  p.tiles = count <= kRankMax ? 0 : static_cast<int>(ceil_div(count, kTile));
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
  bool stream;    // (kCacheBytes)
};

__device__ __forceinline__ void store_zeros(char* p, int64_t bytes, int lane, int lanes, bool stream) {
  // from an address of the element's alignment on; the ends by 2 bytes
  const int64_t head = min<int64_t>(bytes, -reinterpret_cast<intptr_t>(p) & 15);
  const int64_t pieces = (bytes - head) / 16, tail = head + pieces * 16;
  typedef float vec __attribute__((ext_vector_type(4)));
  vec* q = reinterpret_cast<vec*>(p + head);
  const vec zero = {0.0f, 0.0f, 0.0f, 0.0f};
  if (stream)
    for (int64_t i = lane; i < pieces; i += lanes) __builtin_nontemporal_store(zero, q + i);
  else
    for (int64_t i = lane; i < pieces; i += lanes) q[i] = zero;
  for (int64_t i = 2 * lane; i < head; i += 2 * lanes) *reinterpret_cast<uint16_t*>(p + i) = 0;
  for (int64_t i = tail + 2 * lane; i < bytes; i += 2 * lanes) *reinterpret_cast<uint16_t*>(p + i) = 0;
}

template <int NT>
__device__ __forceinline__ void fill_block(const Fill& f, int64_t block) {
  block += f.first;
  if (f.ld_bytes == f.row_bytes) {
    const int64_t from = block * kFillBytes;
    store_zeros(f.dst + from, min<int64_t>(kFillBytes, f.rows * f.row_bytes - from), threadIdx.x, NT, f.stream);
    return;
  }
  const int64_t per = max<int64_t>(1, kFillBytes / f.row_bytes), end = min<int64_t>(f.rows, (block + 1) * per);
  for (int64_t r = block * per + threadIdx.x / kWave; r < end; r += NT / kWave)  // a wave per row
    store_zeros(f.dst + r * f.ld_bytes, f.row_bytes, threadIdx.x % kWave, kWave, f.stream);
}

int64_t fill_blocks(const Fill& f) {
  return f.ld_bytes == f.row_bytes ? ceil_div(f.rows * f.row_bytes, kFillBytes)
                                   : ceil_div(f.rows, std::max<int64_t>(1, kFillBytes / f.row_bytes));
}

__device__ __forceinline__ uint32_t key_at(const ppo_embedding_args& a, int64_t i) {
  const int64_t t = token_at(a.tokens, a.token_type, i, a.vocab);
  return static_cast<uint32_t>(t < 0 ? a.vocab : t);
}

// A block of kRankOwn tokens counts, for each of them, the tokens that come before it in the sorted order: smaller ones, and
// equal ones of a smaller index.  Its waves take 64 of the others at a time, one per lane, and compare them with the own
// tokens, which lie in scalar registers: two instructions each.  The loop is kept short and rolled: as straight-line code of
// ten KB, and with a scalar count of each comparison's bits, it took 14 us for 5,003 tokens, most of it fetching instructions.
// The time goes with count^2, but a sort of as many tokens in one block's LDS leaves the other compute units idle (16 us).
// Four waves: gradients of 5,003 tokens take 22.6 us so, 28.9 with one, 26.0 with two, 25.6 with eight, 32.5 with sixteen (12,000:
// 38.9, 52.5, 45.0, 44.4, 52.5): fewer wait for more loads in a row, more repeat the set-up and the exchanges at the end.
constexpr int kRankThreads = 256, kRankWaves = kRankThreads / kWave, kRankOwn = 16;
static_assert(4 * kRankOwn == kWave, "the reduction's exchanges");
static_assert(kWave % kRankOwn == 0, "a block's tokens lie in one group of 64");

template <class K>  // the tokens' type
__global__ __launch_bounds__(kRankThreads) void rank_kernel(const ppo_embedding_args a, uint32_t* __restrict__ keys,
                                                            uint32_t* __restrict__ idx, int blocks, const Fill fill) {
  __shared__ uint32_t part[kRankWaves][kRankOwn];
  if (static_cast<int>(blockIdx.x) >= blocks) {
    fill_block<kRankThreads>(fill, static_cast<int>(blockIdx.x) - blocks);
    return;
  }
  const int n = static_cast<int>(a.count), groups = (n + kWave - 1) / kWave;
  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int i0 = blockIdx.x * kRankOwn, group = i0 / kWave;
  const K* tokens = static_cast<const K*>(a.tokens);
  auto load = [&](int g) { return tokens[min(g * kWave + lane, n - 1)]; };
  auto key_of = [&](K token, int g) {  // (past the end: before nothing)
    return g * kWave + lane >= n ? INT32_MAX : static_cast<int>(token >= 0 && token < a.vocab ? token : a.vocab);
  };
  const int ours = key_of(load(group), group);
  int own[kRankOwn];
  uint32_t before[kRankOwn];
#pragma unroll
  for (int t = 0; t < kRankOwn; ++t) {
    own[t] = __builtin_amdgcn_readlane(ours, i0 % kWave + t);
    before[t] = 0;
  }
  if (wave == group % kRankWaves) {  // the own group: by index where equal
#pragma unroll
    for (int t = 0; t < kRankOwn; ++t) before[t] = ours < own[t] + (lane < i0 % kWave + t ? 1 : 0) ? 1 : 0;
  }
  // four groups' loads ahead of the comparisons (tokens as they are: a key made of one would wait for it)
  K next[4];
#pragma unroll
  for (int f = 0; f < 4; ++f) next[f] = load(wave + f * kRankWaves);
#pragma unroll 1
  for (int g0 = wave; g0 < groups; g0 += 4 * kRankWaves)
#pragma unroll
    for (int f = 0; f < 4; ++f) {
      const int g = g0 + f * kRankWaves;
      const int key = key_of(next[f], g);
      const int theirs = g < group ? key - 1 : g > group ? key : INT32_MAX;  // (x <= y as x - 1 < y)
      next[f] = load(g + 4 * kRankWaves);
#pragma unroll
      for (int t = 0; t < kRankOwn; ++t) before[t] += theirs < own[t] ? 1 : 0;
    }
  // the lanes' counts: with each exchange a lane keeps half of the tokens, until it holds one of them over 4 lanes
#pragma unroll
  for (int d = kWave / 2, half = kRankOwn / 2; half > 0; d /= 2, half /= 2)
#pragma unroll
    for (int t = 0; t < half; ++t) {
      const uint32_t send = lane & d ? before[t] : before[t + half], keep = lane & d ? before[t + half] : before[t];
      before[t] = keep + __shfl_xor(send, d, kWave);
    }
  before[0] += __shfl_xor(before[0], 2, kWave);
  before[0] += __shfl_xor(before[0], 1, kWave);
  if (lane % 4 == 0) part[wave][lane / 4] = before[0];
  __syncthreads();
  if (threadIdx.x >= kRankOwn || i0 + lane >= n) return;
  uint32_t to = 0;
  int key = 0;
#pragma unroll
  for (int w = 0; w < kRankWaves; ++w) to += part[w][lane];
#pragma unroll
  for (int t = 0; t < kRankOwn; ++t) key = lane == t ? own[t] : key;
  keys[to] = key;
  idx[to] = i0 + lane;
}

__device__ __forceinline__ int item_in_tile(int round) {
  return (threadIdx.x / kWave) * (kRounds * kWave) + round * kWave + (threadIdx.x & (kWave - 1));
}

// Stable ranks of a tile's digits: rank[r] counts the items of the same digit before this one in its wave, and
// counts[wave][digit] becomes how many the wave holds.  counts is zero on entry.  The lanes of a digit find each other by a
// ballot per bit.
__device__ __forceinline__ void wave_ranks(const uint32_t (&digit)[kRounds], const bool (&in)[kRounds], int bits,
                                           uint32_t* counts, uint32_t (&rank)[kRounds]) {
  uint32_t* mine = counts + (threadIdx.x / kWave) * kMaxDigits;
  const uint64_t below = (uint64_t{1} << (threadIdx.x & (kWave - 1))) - 1;
  uint64_t same[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) same[r] = __ballot(in[r]);
#pragma unroll
  for (int b = 0; b < kMaxBits; ++b)
    if (b < bits) {
#pragma unroll
      for (int r = 0; r < kRounds; ++r) {
        const bool set = (digit[r] >> b) & 1;
        const uint64_t m = __ballot(set);
        same[r] &= set ? m : ~m;
      }
    }
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
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

// One pass over several tiles: how many items of each digit a tile holds, hist[tile][digit]; then every item to its place.
__global__ __launch_bounds__(kSortThreads) void sort_count_kernel(const ppo_embedding_args a, int shift, int bits, int tiles,
                                                                  const uint32_t* __restrict__ keys,
                                                                  uint32_t* __restrict__ hist, const Fill fill) {
  __shared__ uint32_t count[kMaxDigits];
  if (static_cast<int>(blockIdx.x) >= tiles) {
    fill_block<kSortThreads>(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
  const int64_t base = static_cast<int64_t>(blockIdx.x) * kTile;
  uint32_t key[kRounds];
#pragma unroll
  for (int r = 0; r < kRounds; ++r) {
    const int64_t i = base + r * kSortThreads + threadIdx.x;
    key[r] = i < a.count ? (keys != nullptr ? keys[i] : key_at(a, i)) : 0;
  }
  if (threadIdx.x < kMaxDigits) count[threadIdx.x] = 0;
  __syncthreads();
#pragma unroll
  for (int r = 0; r < kRounds; ++r)
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
    fill_block<kSortThreads>(fill, static_cast<int>(blockIdx.x) - tiles);
    return;
  }
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
  for (int r = 0; r < kRounds; ++r)
    if (in[r]) {
      const uint32_t to = start[digit[r]] + counts[(threadIdx.x / kWave) * kMaxDigits + digit[r]] + rank[r];
      keys[to] = key[r];
      idx[to] = from[r];
    }
}

// ---- the sums ----

// 131,072 bf16 rows of 1,024 into 65,536 fp32 rows: 74 us, 274 MB read and 118 written, 5.3 TB/s; the joins 12, the sort with the
// zeros 53.
// The sorted positions are cut into units; a wave sums a unit's rows over 64 16-byte pieces of columns.  A run of one token
// that crosses into the next unit by at most kReach rows is finished where it began, and the next unit starts behind it.  A run
// that goes on further leaves its parts in `partial` ([units][2][dim]: of the run that came into the unit, of the one that goes
// out), joined by embedding_join_kernel in the units' order.
constexpr int kFlight = 8;                    // rows' loads a wave issues together; it has two such groups in flight
constexpr uint32_t kReach = 8, kMaxUnit = 32;  // (a unit, what it reaches and one more position fit a wave's lanes)
static_assert(kMaxUnit + kReach < kWave, "a unit's keys, one per lane");

struct SumArgs {
  ppo_embedding_args e;
  const uint32_t* keys;
  const uint32_t* idx;
  float* partial;
  int64_t ld_partial;  // a multiple of 4
  uint32_t unit;       // positions, kReach to kMaxUnit
  uint32_t units;
  uint32_t columns;    // waves side by side on a row
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
  constexpr uint32_t kNone = 0xffffffffu;  // no key
  const ppo_embedding_args& a = s.e;
  const uint32_t lane = threadIdx.x, n = static_cast<uint32_t>(a.count);
  const uint32_t unit = blockIdx.x / s.columns, column = blockIdx.x % s.columns, begin = unit * s.unit;  // a row's parts at about one time
  // each lane a position's key and index, from the unit's first on
  const uint32_t at = begin + lane;
  const uint32_t keys = at < n ? s.keys[at] : kNone, idx = at < n ? s.idx[at] : 0;
  const uint32_t before = begin > 0 ? s.keys[begin - 1] : kNone;
  auto key_of = [&](uint32_t i) { return static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(keys), static_cast<int>(i))); };
  auto run_from = [&](uint32_t i, uint32_t key) {  // how many positions from the i-th on hold the key
    const uint64_t other = __ballot(keys != key) >> i;
    return other == 0 ? kWave - i : static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(other)) - 1);
  };
  uint32_t first = 0, last = min(s.unit, n - begin);  // the positions this wave sums, from `begin` on
  bool head = false, tail = false;                    // the first run came in, the last one goes on
  if (begin > 0) {
    first = run_from(0, before);
    head = first > kReach;
    if (head) first = 0;
  }
  const uint32_t more = last < s.unit ? 0 : run_from(last, key_of(last - 1));
  tail = more > kReach;
  if (!tail) last += more;
  if (first >= last) return;  // the unit before has taken all of it

  O* out = static_cast<O*>(a.dst);
  const int c0 = static_cast<int>(column * kWave + lane) * V;
  const bool whole = a.dim >= V;
  const int c = whole ? min(c0, a.dim - V) : 0;  // an odd row's last piece is read from V columns before its end
  const T* src = static_cast<const T*>(a.src);
  uint32_t cur = key_of(first);
  float sum[V] = {};
  auto flush = [&](bool part) {
    if (cur < a.vocab) {
      if (part)
        store_sum<V>(s.partial + (static_cast<int64_t>(unit) * 2 + (head ? 0 : 1)) * s.ld_partial, c0, c, a.dim, sum, 1.0f, false);
      else
        store_sum<V>(out + static_cast<int64_t>(cur) * a.ld_dst, c0, c, a.dim, sum, a.scale, a.accumulate != 0);
    }
    head = false;
#pragma unroll
    for (int i = 0; i < V; ++i) sum[i] = 0.0f;
  };
  struct Group {
    typename Piece<T>::type x[kFlight];
  };
  auto load = [&](Group& g, uint32_t p) {
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      const int64_t i = static_cast<uint32_t>(__builtin_amdgcn_readlane(static_cast<int>(idx), static_cast<int>(min(p + u, last - 1))));
      const T* row = src + i * a.ld_src;
      if (whole) {
        g.x[u] = load_piece<true>(row + c);  // (read once)
      } else {
#pragma unroll
        for (int e = 0; e < V; ++e) g.x[u][e] = e < a.dim ? row[e] : static_cast<T>(0.0f);
      }
    }
  };
  auto add = [&](const Group& g, uint32_t p) {
#pragma unroll
    for (int u = 0; u < kFlight; ++u) {
      if (p + u >= last) break;
      const uint32_t key = key_of(p + u);
      if (key != cur) {
        flush(head);
        cur = key;
      }
      const typename Piece<T>::type x = g.x[u];
#pragma unroll
      for (int i = 0; i < V; ++i) sum[i] += static_cast<float>(x[i]);
    }
  };
  // the next group's loads go out before this one's sums and their stores, whose completion they then need not wait for
  Group even, odd;
  load(even, first);
  for (uint32_t p = first; p < last; p += 2 * kFlight) {
    if (p + kFlight < last) load(odd, p + kFlight);
    add(even, p);
    if (p + 2 * kFlight < last) load(even, p + 2 * kFlight);
    if (p + kFlight < last) add(odd, p + kFlight);
  }
  flush(head || tail);
}

// The runs that go on past a unit by more than kReach: a wave per unit adds the parts of those that begin there, unless there
// are so many that the block's waves share them (at most one such run can begin in a block's units).
constexpr int kJoinWaves = 16, kJoinThreads = kJoinWaves * kWave, kJoinColumns = 4 * kWave;
constexpr uint32_t kJoinAlone = 16;

template <class O>
__global__ __launch_bounds__(kJoinThreads) void embedding_join_kernel(const SumArgs s) {
  __shared__ float4 part[kJoinWaves][kWave];
  __shared__ uint32_t shared_unit, shared_more;
  const ppo_embedding_args& a = s.e;
  const uint32_t n = static_cast<uint32_t>(a.count), lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
  const uint32_t u = blockIdx.x * kJoinWaves + wave;
  // whether a run goes on past the boundary before position b: the position kReach behind it still holds its key
  auto crosses = [&](uint64_t b, uint32_t key) { return b + kReach < n && s.keys[b + kReach] == key; };
  const uint64_t begin = static_cast<uint64_t>(u) * s.unit, end = begin + s.unit;
  uint32_t key = 0, more = 0;  // the units that the run goes on in
  if (end + kReach < n) {
    key = s.keys[end - 1];
    const uint32_t behind = s.keys[end + kReach], before = begin > 0 ? s.keys[begin - 1] : ~0u;
    if (behind == key && key < a.vocab && before != key) {
      // 64 boundaries at once; of a longer run every 64th first
      auto leading = [&](uint32_t from, uint32_t step) {
        const uint64_t m = __ballot(crosses(end + static_cast<uint64_t>(from + lane * step) * s.unit, key));
        return m == ~uint64_t{0} ? static_cast<uint32_t>(kWave) : static_cast<uint32_t>(__ffsll(static_cast<unsigned long long>(~m)) - 1);
      };
      more = leading(0, 1);
      if (more == kWave) {
        uint32_t far = 0;
        for (uint32_t k = kWave; k == kWave; far += k) k = leading(far * kWave, kWave);
        more = (far - 1) * kWave;
        more += leading(more, 1);
      }
    }
  }
  const int c = (blockIdx.y * kWave + static_cast<int>(lane)) * 4;
  auto sum_of = [&](uint32_t unit, uint32_t from, uint32_t to) {  // the parts of units unit + from .. unit + to - 1
    float4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (c < a.dim) {
#pragma unroll 8
      for (uint32_t i = from; i < to; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(s.partial + (static_cast<int64_t>(unit + i) * 2 + (i == 0 ? 1 : 0)) * s.ld_partial + c);
        sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
      }
    }
    return sum;
  };
  auto store = [&](uint32_t row, const float4& sum) {
    const float x[4] = {sum.x, sum.y, sum.z, sum.w};
    O* to = static_cast<O*>(a.dst) + static_cast<int64_t>(row) * a.ld_dst + c;
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (c + i < a.dim) to[i] = static_cast<O>(a.accumulate ? static_cast<float>(to[i]) + a.scale * x[i] : a.scale * x[i]);
  };
  if (threadIdx.x == 0) shared_more = 0;
  __syncthreads();
  if (more > kJoinAlone && lane == 0) {
    shared_unit = u;
    shared_more = more;
  }
  if (more > 0 && more <= kJoinAlone) store(key, sum_of(u, 0, more + 1));
  __syncthreads();
  const uint32_t all = shared_more + 1;
  if (all == 1) return;
  const uint32_t share = (all + kJoinWaves - 1) / kJoinWaves;
  part[wave][lane] = sum_of(shared_unit, min(all, wave * share), min(all, (wave + 1) * share));
  __syncthreads();
  if (u != shared_unit) return;
  float4 sum = part[0][lane];
#pragma unroll
  for (int w = 1; w < kJoinWaves; ++w) {
    const float4 x = part[w][lane];
    sum.x += x.x, sum.y += x.y, sum.z += x.z, sum.w += x.w;
  }
  store(key, sum);
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

int check_apart(const char* who, const ppo_embedding_args& a, bool bwd) {
  const int64_t in = type_size(a.src_type), out = type_size(a.dst_type);
  const Rows src{a.src, bwd ? a.count : a.vocab, a.dim * in, a.ld_src * in}, dst{a.dst, bwd ? a.vocab : a.count, a.dim * out, a.ld_dst * out};
  const Rows tokens = vector_of(a.tokens, a.count * (a.token_type == PPO_TOKENS_I64 ? 8 : 4));
  PPO_REQUIRE(a.count == 0 || !(overlap(dst, src) || overlap(dst, tokens)), "%s: dst overlaps an input", who);
  return PPO_OK;
}

struct BwdLayout {
  SortPlan sort;
  uint32_t unit, units;
  int64_t ld_partial;
  size_t keys[2], idx[2], hist, partial, bytes;
};

// Positions of a unit: enough waves to fill the chip (16 KiB of loads in flight each), but no fewer than a run may reach past its
// unit.
uint32_t unit_for(int64_t count, int32_t dim) {
  const int64_t waves = count * ceil_div(dim, 512);  // of one position each (of 16-bit rows; the workspace goes by it too)
  if (count <= kMaxUnit) return kMaxUnit;  // one unit, nothing to join
  uint32_t unit = kReach;
  while (unit < kMaxUnit && waves > static_cast<int64_t>(unit) * 8192) unit *= 2;
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
  l.hist = take(l.sort.tiles > 0 ? 4 * static_cast<size_t>(l.sort.digits()) * l.sort.tiles : 0);
  l.partial = take(8 * static_cast<size_t>(l.units) * l.ld_partial);
  l.bytes = at;
  return l;
}

template <class T, class O>
int launch_sums(SumArgs s, hipStream_t st) {
  const int dim = s.e.dim;
  s.columns = static_cast<uint32_t>(ceil_div(dim, kWave * kVec<T>));
  PPO_REQUIRE(static_cast<int64_t>(s.units) * s.columns < INT32_MAX, "ppo_embedding_bwd: count=%lld dim=%d", (long long)s.e.count, dim);
  hipLaunchKernelGGL((embedding_sum_kernel<T, O>), dim3(s.units * s.columns), dim3(kWave), 0, st, s);
  if (int rc = check_launch("embedding_sum_kernel")) return rc;
  if (s.units < 2) return PPO_OK;
  const dim3 join(static_cast<uint32_t>(ceil_div(s.units, kJoinWaves)), static_cast<uint32_t>(ceil_div(dim, kJoinColumns)));
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
  if (int rc = check_apart("ppo_embedding_fwd", a, false)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = PPO_OK;
  with_type(a.src_type, [&](auto t) {
    using T = decltype(t);
    const int64_t pieces = ceil_div(a.dim, kVec<T>);
    int log_tpr = 0;
    while ((1 << log_tpr) < pieces && (1 << log_tpr) < kFwdThreads) ++log_tpr;
    const int64_t blocks = ceil_div(a.count, static_cast<int64_t>(kFwdThreads >> log_tpr) * kFwdRows);
    const dim3 grid(static_cast<uint32_t>(std::min(blocks, kFwdGrid)), static_cast<uint32_t>(ceil_div(pieces, 1 << log_tpr)),
                    static_cast<uint32_t>(ceil_div(blocks, kFwdGrid)));
    hipLaunchKernelGGL(embedding_fwd_kernel<T>, grid, dim3(kFwdThreads), 0, st, a, log_tpr);
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
  if (int rc = check_apart("ppo_embedding_bwd", a, true)) return rc;
  if (a.count == 0 && a.accumulate) return PPO_OK;
  hipStream_t st = static_cast<hipStream_t>(stream);
  char* ws = static_cast<char*>(workspace);
  auto at = [&](size_t offset) { return reinterpret_cast<uint32_t*>(ws + offset); };
  const int64_t size = type_size(a.dst_type);
  Fill fill{static_cast<char*>(a.dst), a.vocab, a.dim * size, a.ld_dst * size, 0,
            (a.vocab * size + a.count * type_size(a.src_type)) * a.dim > kCacheBytes};
  const int64_t blocks = a.accumulate ? 0 : fill_blocks(fill);
  PPO_REQUIRE(blocks < (int64_t{1} << 30), "ppo_embedding_bwd: the table is too large");
  int last = 0;  // the buffer that holds the sorted tokens
  if (l.sort.tiles == 0) {
    const int own = static_cast<int>(ceil_div(a.count, kRankOwn));
    const dim3 grid(own + static_cast<uint32_t>(blocks));
    if (a.token_type == PPO_TOKENS_I64)
      hipLaunchKernelGGL(rank_kernel<int64_t>, grid, dim3(kRankThreads), 0, st, a, at(l.keys[0]), at(l.idx[0]), own, fill);
    else
      hipLaunchKernelGGL(rank_kernel<int32_t>, grid, dim3(kRankThreads), 0, st, a, at(l.keys[0]), at(l.idx[0]), own, fill);
    if (int rc = check_launch("rank_kernel")) return rc;
    if (a.count == 0) return PPO_OK;
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
  const SumArgs s{a, at(l.keys[last]), at(l.idx[last]), reinterpret_cast<float*>(ws + l.partial), l.ld_partial, l.unit, l.units, 0};
  int rc = PPO_OK;
  with_type(a.src_type, [&](auto t) {
    using T = decltype(t);
    if (a.dst_type == PPO_TYPE_F32) rc = launch_sums<T, float>(s, st);
    else rc = launch_sums<T, T>(s, st);
  });
  return rc;
}
