// Queries and keys of each head normed and turned by their token's position, and the gradients (ppo_qk_rotary_fwd, _bwd).
//
// A row (one head of one token) is D / 2 pairs: pair i < R / 2 is turned by positions[token] freqs[i]; what the rotation leaves out is
// paired up too (i with i + (D - R) / 2) and turned by nothing, so that every lane does the same: it holds V pairs as two pieces of V
// elements and needs no other lane but for the row's sums.  LANES lanes, a power of two, hold a row.
//   y = x r w turned, r = 1 / sqrt(sum x^2 / D + eps);
//   going back, g = dy turned back:   dw += g x r;   dx = r (g w - x r^2 sum(g w x) / D).
// Angles: positions * freqs in fp64, as turns less the nearest whole number; the fraction is exact enough in fp32 for sincospi, however
// far the position.  A block takes the sines and cosines of its tokens once, for all its heads, into LDS.
//
// Bound by memory: x once in, y once out (dx: x and dy in).  Weight gradients stay in registers over a block's tokens (and, where heads
// share the weight, over its heads), then go to the workspace, and a last launch adds the blocks' in a fixed order in fp64.
// 16,384 tokens of 24 heads of 128 (201 MB in and out): 37 us, the copy's rate; going back 32,768 tokens of 24 heads of 128 (604 MB): 132 us, 4.6 TB/s (144 with a
// head's tokens one after another, whose rows lie apart, where the heads share a weight), and 5 for the join: a row's sums have to be there before it is
// written, and few of a wave's rows are on their way meanwhile.
#include "views.hpp"

namespace ppo {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kTurns = 4096;  // sines and cosines that a block holds at most: 32 KB of LDS
constexpr int kMaxTile = 64;  // tokens of a block at most
constexpr int kMostSummed = 512;  // rows of a sum in fp32

struct QkArgs {
  ppo_qk_rotary_args a;
  float* partial;     // [tiles][heads, or 2][D], backward
  int32_t tile;       // tokens of a block
  int32_t group;      // heads of a block
  int32_t lanes_log2; // of a row
  float inv_dim, eps;
};

template <class R>
__device__ __forceinline__ R row_sum(R x, int lanes) {
  for (int d = lanes / 2; d > 0; d >>= 1) x += __shfl_xor(x, d, kWave);
  return x;
}

// A view's row of one head and token.
template <class T>
__device__ __forceinline__ T* row_at(const ppo_head_view& v, int64_t token, int head) {
  return static_cast<T*>(v.data) + token * v.token_stride + head * v.head_stride;
}

// Where a unit of V pairs starting at pair p lies in its row: two pieces of V elements each, or with interleaved pairs 2 V neighbours.
struct Place {
  int a, b;
  bool neighbours, turned;
};
__device__ __forceinline__ Place place_of(const ppo_qk_rotary_args& a, int p) {
  const int half = a.rotary_dim / 2;
  Place o;
  o.turned = p < half;
  o.neighbours = o.turned && a.interleaved != 0;
  if (o.neighbours) o.a = 2 * p, o.b = 2 * p;
  else if (o.turned) o.a = p, o.b = p + half;
  else o.a = half + p, o.b = half + p + (a.head_dim / 2 - half);
  return o;
}

template <class T, int V>
__device__ __forceinline__ void load_pairs(const T* row, const Place& at, float (&x)[V], float (&y)[V]) {
  typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if constexpr (V == 1) {
    x[0] = static_cast<float>(row[at.a]);
    y[0] = static_cast<float>(row[at.neighbours ? at.a + 1 : at.b]);
  } else {
    const Vec u = *reinterpret_cast<const Vec*>(row + at.a), v = *reinterpret_cast<const Vec*>(row + (at.neighbours ? at.a + V : at.b));
    float f[2 * V];
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = static_cast<float>(u[i]), f[V + i] = static_cast<float>(v[i]);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      x[i] = at.neighbours ? f[2 * i] : f[i];
      y[i] = at.neighbours ? f[2 * i + 1] : f[V + i];
    }
  }
}

template <class T, int V>
__device__ __forceinline__ void store_pairs(T* row, const Place& at, const float (&x)[V], const float (&y)[V]) {
  typedef T Vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  if constexpr (V == 1) {
    row[at.a] = static_cast<T>(x[0]);
    row[at.neighbours ? at.a + 1 : at.b] = static_cast<T>(y[0]);
  } else {
    Vec u, v;
    if (at.neighbours) {
#pragma unroll
      for (int i = 0; i < V / 2; ++i) {
        u[2 * i] = static_cast<T>(x[i]), u[2 * i + 1] = static_cast<T>(y[i]);
        v[2 * i] = static_cast<T>(x[V / 2 + i]), v[2 * i + 1] = static_cast<T>(y[V / 2 + i]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) u[i] = static_cast<T>(x[i]), v[i] = static_cast<T>(y[i]);
    }
    *reinterpret_cast<Vec*>(row + at.a) = u;
    *reinterpret_cast<Vec*>(row + (at.neighbours ? at.a + V : at.b)) = v;
  }
}

// Sines and cosines of the block's tokens and of every turned pair, [token][pair].
__device__ __forceinline__ void fill_turns(const QkArgs& q, int64_t first, int count, float2* turns) {
  const int half = q.a.rotary_dim / 2;
  for (int i = threadIdx.x; i < count * half; i += kThreads) {
    const int64_t t = first + i / half;
    const int64_t pos = q.a.position_type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(q.a.positions)[t]
                                                            : static_cast<int64_t>(static_cast<const int32_t*>(q.a.positions)[t]);
    const double whole = static_cast<double>(pos) * q.a.freqs[i % half] * 0.15915494309189533577;  // 1 / (2 pi)
    float s, c;
    sincospif(2.0f * static_cast<float>(whole - rint(whole)), &s, &c);
    turns[i] = make_float2(c, s);
  }
  __syncthreads();
}

template <class T, int V>
__device__ __forceinline__ void load_weight(const QkArgs& q, const void* weight, int head, const Place& at, float (&x)[V], float (&y)[V]) {
  const int64_t off = q.a.weight_per_head != 0 ? static_cast<int64_t>(head) * q.a.head_dim : 0;
  if (sizeof(T) == 4 || q.a.weight_type != PPO_TYPE_F32) load_pairs<T, V>(static_cast<const T*>(weight) + off, at, x, y);
  else load_pairs<float, V>(static_cast<const float*>(weight) + off, at, x, y);
}

// A block: a tile of tokens, a group of heads (queries' first, then keys').  UNITS: units of V pairs that a lane holds.
template <class T, int V, int UNITS>
__global__ __launch_bounds__(kThreads) void qk_rotary_kernel(const QkArgs q) {
  __shared__ float2 turns[kTurns];
  const int half = q.a.rotary_dim / 2, pairs = q.a.head_dim / 2, lanes = 1 << q.lanes_log2;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * q.tile;
  const int count = static_cast<int>(min(static_cast<int64_t>(q.tile), q.a.tokens - first));
  const int head0 = blockIdx.y * q.group, heads = min(q.group, q.a.q_heads + q.a.kv_heads - head0);
  fill_turns(q, first, count, turns);
  const int lane = threadIdx.x & (lanes - 1);
  for (int row = threadIdx.x >> q.lanes_log2; row < count * heads; row += kThreads >> q.lanes_log2) {
    const int t = row / heads, h = head0 + row % heads;
    const bool key = h >= q.a.q_heads;
    const int head = key ? h - q.a.q_heads : h;
    const T* x = row_at<const T>(key ? q.a.k : q.a.q, first + t, head);
    float xa[UNITS][V], xb[UNITS][V], sum = 0.0f;
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int p = (lane + u * lanes) * V;
      if (p < pairs) {
        load_pairs<T, V>(x, place_of(q.a, p), xa[u], xb[u]);
#pragma unroll
        for (int e = 0; e < V; ++e) sum = fmaf(xa[u][e], xa[u][e], fmaf(xb[u][e], xb[u][e], sum));
      }
    }
    const float r = 1.0f / sqrtf(row_sum(sum, lanes) * q.inv_dim + q.eps);
    T* y = row_at<T>(key ? q.a.k_out : q.a.q_out, first + t, head);
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int p = (lane + u * lanes) * V;
      if (p < pairs) {
        const Place at = place_of(q.a, p);
        float wa[V], wb[V];
        load_weight<T, V>(q, key ? q.a.k_weight : q.a.q_weight, head, at, wa, wb);
#pragma unroll
        for (int e = 0; e < V; ++e) {
          const float a = xa[u][e] * r * wa[e], b = xb[u][e] * r * wb[e];
          const float2 cs = at.turned ? turns[t * half + p + e] : make_float2(1.0f, 0.0f);
          xa[u][e] = at.turned ? a * cs.x - b * cs.y : a;  // (a value that is not finite stays out of its neighbour's, as in the formula)
          xb[u][e] = at.turned ? b * cs.x + a * cs.y : b;
        }
        store_pairs<T, V>(y, at, xa[u], xb[u]);
      }
    }
  }
}

// Backward.  The block's waves share each head's tokens; a weight gradient leaves the registers at the end of a head (weight_per_head)
// or of the queries' or keys' heads.
template <class T, int V, int UNITS>
__global__ __launch_bounds__(kThreads) void qk_rotary_bwd_kernel(const QkArgs q) {
  __shared__ float2 turns[kTurns];
  __shared__ float joined[kWaves][PPO_QK_MAX_DIM];
  const int half = q.a.rotary_dim / 2, pairs = q.a.head_dim / 2, lanes = 1 << q.lanes_log2, dim = q.a.head_dim;
  const int64_t first = static_cast<int64_t>(blockIdx.x) * q.tile;
  const int count = static_cast<int>(min(static_cast<int64_t>(q.tile), q.a.tokens - first));
  const int all = q.a.q_heads + q.a.kv_heads, head0 = blockIdx.y * q.group, heads = min(q.group, all - head0);
  const bool per_head = q.a.weight_per_head != 0;
  fill_turns(q, first, count, turns);
  const int lane = threadIdx.x & (lanes - 1);
  float da[UNITS][V] = {}, db[UNITS][V] = {};
  for (int h = head0, next; h < head0 + heads; h = next) {
    // one head, or all that share a weight: then rows in the order in which they lie
    const bool key = h >= q.a.q_heads;
    next = per_head ? h + 1 : key ? head0 + heads : min(head0 + heads, q.a.q_heads);
    const int together = next - h;
    for (int i = threadIdx.x >> q.lanes_log2; i < count * together; i += kThreads >> q.lanes_log2) {
      const int t = together == 1 ? i : i / together, head = (key ? h - q.a.q_heads : h) + i - t * together;
      const T* x = row_at<const T>(key ? q.a.k : q.a.q, first + t, head);
      const T* dy = row_at<const T>(key ? q.a.k_out : q.a.q_out, first + t, head);
      float xa[UNITS][V], xb[UNITS][V], ga[UNITS][V], gb[UNITS][V], sum = 0.0f, dot = 0.0f;
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int p = (lane + u * lanes) * V;
        if (p < pairs) {
          const Place at = place_of(q.a, p);
          load_pairs<T, V>(x, at, xa[u], xb[u]);
          load_pairs<T, V>(dy, at, ga[u], gb[u]);
          float wa[V], wb[V];
          load_weight<T, V>(q, key ? q.a.k_weight : q.a.q_weight, head, at, wa, wb);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 cs = at.turned ? turns[t * half + p + e] : make_float2(1.0f, 0.0f);
            const float a = at.turned ? ga[u][e] * cs.x + gb[u][e] * cs.y : ga[u][e];
            const float b = at.turned ? gb[u][e] * cs.x - ga[u][e] * cs.y : gb[u][e];
            ga[u][e] = a, gb[u][e] = b;
            sum = fmaf(xa[u][e], xa[u][e], fmaf(xb[u][e], xb[u][e], sum));
            dot = fmaf(a * wa[e], xa[u][e], fmaf(b * wb[e], xb[u][e], dot));
          }
        }
      }
      const float r = 1.0f / sqrtf(row_sum(sum, lanes) * q.inv_dim + q.eps);
      const float c = row_sum(dot, lanes) * r * q.inv_dim * r;  // n c' = x r (r sum(g w x) / D)
      T* dx = row_at<T>(key ? q.a.d_k : q.a.d_q, first + t, head);
#pragma unroll
      for (int u = 0; u < UNITS; ++u) {
        const int p = (lane + u * lanes) * V;
        if (p < pairs) {
          const Place at = place_of(q.a, p);
          float wa[V], wb[V];
          load_weight<T, V>(q, key ? q.a.k_weight : q.a.q_weight, head, at, wa, wb);
#pragma unroll
          for (int e = 0; e < V; ++e) {
            da[u][e] = fmaf(ga[u][e], xa[u][e] * r, da[u][e]);
            db[u][e] = fmaf(gb[u][e], xb[u][e] * r, db[u][e]);
            xa[u][e] = r * (ga[u][e] * wa[e] - xa[u][e] * c);
            xb[u][e] = r * (gb[u][e] * wb[e] - xb[u][e] * c);
          }
          store_pairs<T, V>(dx, at, xa[u], xb[u]);
        }
      }
    }
    // lanes of the same pairs, then waves, in order
#pragma unroll
    for (int u = 0; u < UNITS; ++u) {
      const int p = (lane + u * lanes) * V;
      const Place at = place_of(q.a, min(p, pairs - V));
#pragma unroll
      for (int e = 0; e < V; ++e) {
        float sa = da[u][e], sb = db[u][e];
        for (int d = lanes; d < kWave; d <<= 1) sa += __shfl_xor(sa, d, kWave), sb += __shfl_xor(sb, d, kWave);
        if (p < pairs && threadIdx.x % kWave < lanes) {
          joined[threadIdx.x / kWave][at.neighbours ? at.a + 2 * e : at.a + e] = sa;
          joined[threadIdx.x / kWave][at.neighbours ? at.a + 2 * e + 1 : at.b + e] = sb;
        }
        da[u][e] = db[u][e] = 0.0f;
      }
    }
    __syncthreads();
    const int slot = per_head ? h : (key ? 1 : 0), slots = per_head ? all : 2;
    // (a group of heads that share a weight adds to its tile's row of its own: tiles * groups rows)
    const int64_t row = per_head ? blockIdx.x : static_cast<int64_t>(blockIdx.x) * gridDim.y + blockIdx.y;
    float* out = q.partial + (row * slots + slot) * dim;
    for (int i = threadIdx.x; i < dim; i += kThreads) out[i] = (joined[0][i] + joined[1][i]) + (joined[2][i] + joined[3][i]);
    if (!per_head) {  // the side that a group of heads does not touch
      const bool other = key ? head0 >= q.a.q_heads : head0 + heads <= q.a.q_heads;
      if (other)
        for (int i = threadIdx.x; i < dim; i += kThreads) q.partial[(row * slots + (1 - slot)) * dim + i] = 0.0f;
    }
    __syncthreads();
  }
}

// The blocks' sums of 16 elements of one weight gradient: each of 64 rows of lanes adds every 64th block's, then these are added.  (Blocks of 64 elements, 16 rows
// of lanes: 12 us for 1,024 tiles' 2 x 128 elements, four blocks, so 5.)
constexpr int kJoinThreads = 1024, kJoinWidth = 16, kJoinRows = kJoinThreads / kJoinWidth;
template <class W>
__global__ __launch_bounds__(kJoinThreads) void qk_rotary_join_kernel(const QkArgs q, int64_t rows) {
  __shared__ double part[kJoinRows][kJoinWidth];
  const bool per_head = q.a.weight_per_head != 0;
  const int dim = q.a.head_dim, slots = per_head ? q.a.q_heads + q.a.kv_heads : 2, slot = blockIdx.y;
  const int column = threadIdx.x % kJoinWidth, mine = threadIdx.x / kJoinWidth, i = blockIdx.x * kJoinWidth + column;
  double sum = 0.0;
  constexpr int AHEAD = 8;  // loads in flight
  if (i < dim)
    for (int64_t r = mine; r < rows; r += kJoinRows * AHEAD) {
      float x[AHEAD];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) x[u] = q.partial[(min(r + u * kJoinRows, rows - 1) * slots + slot) * dim + i];
#pragma unroll
      for (int u = 0; u < AHEAD; ++u) sum += r + u * kJoinRows < rows ? static_cast<double>(x[u]) : 0.0;
    }
  part[mine][column] = sum;
  for (int n = kJoinRows / 2; n > 0; n /= 2) {  // (in pairs: the same order every time)
    __syncthreads();
    if (mine < n) part[mine][column] = sum += part[mine + n][column];
  }
  if (mine != 0 || i >= dim) return;
  const bool key = per_head ? slot >= q.a.q_heads : slot == 1;
  W* out = static_cast<W*>(key ? q.a.d_k_weight : q.a.d_q_weight);
  const int head = per_head ? (key ? slot - q.a.q_heads : slot) : 0;
  out[head * dim + i] = static_cast<W>(static_cast<float>(sum));
}

constexpr int64_t kMostTokens = (int64_t{1} << 28) - 16;  // 16 a block: a launch holds fewer than 2^32 threads

struct Plan {
  int vec, units, lanes_log2, tile, group;
  int64_t tiles, groups, rows, slots;  // rows: of partial sums
};

Plan plan_of(const ppo_qk_rotary_args& a, bool backward) {
  Plan p{};
  const int pairs = a.head_dim / 2, half = a.rotary_dim / 2, whole = a.type == PPO_TYPE_F32 ? 4 : 8;
  p.vec = pairs % whole == 0 && half % whole == 0 ? whole : 1;
  const int units = pairs / p.vec;
  while ((1 << p.lanes_log2) < units && p.lanes_log2 < 6) ++p.lanes_log2;
  p.units = static_cast<int>(ceil_div(units, 1 << p.lanes_log2));
  if (p.units == 3) p.units = 4;
  const int heads = a.q_heads + a.kv_heads, at_once = kThreads >> p.lanes_log2;
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  // Tokens of a block: as many as share the sines, but blocks enough for the chip; going back, where a block takes a head's tokens at a time, as many
  // as it has rows for at least (4,099 tokens of 8 heads of 80, a weight each: 4 tokens a block 40 us, 16 and a head a block 15).
  p.tile = std::min(kMaxTile, std::max(1, kTurns / std::max(1, half)));
  if (!backward) p.tile = std::min(p.tile, 16);
  const int least = backward ? std::min(p.tile, at_once) : 1;
  while (p.tile > least && ceil_div(a.tokens, p.tile) < 4 * cus) p.tile = std::max(least, p.tile / 2);
  p.tiles = ceil_div(a.tokens, p.tile);
  // heads of a block: all, which share the sines (512 tokens of 20 heads of 128: 3.9 us, 5 a block 5.8), unless that leaves the chip idle: more than a block has
  // rows for, or going back
  p.group = heads;
  while (p.group > 1 && p.tiles * ceil_div(heads, p.group) < 4 * cus && (backward || p.group * p.tile > at_once)) p.group = (p.group + 1) / 2;
  // (going back a lane adds up every at_once-th row of its block before they go on in fp64)
  if (backward && a.weight_per_head == 0) p.group = std::min(p.group, std::max(1, kMostSummed * at_once / p.tile));
  p.groups = ceil_div(heads, p.group);
  p.rows = a.weight_per_head != 0 ? p.tiles : p.tiles * p.groups;
  p.slots = a.weight_per_head != 0 ? heads : 2;
  return p;
}

int check(const char* who, const ppo_qk_rotary_args* args, bool backward) {
  PPO_REQUIRE(args != nullptr, "%s: null arguments", who);
  const ppo_qk_rotary_args& a = *args;
  PPO_REQUIRE(a.tokens >= 0 && a.tokens < kMostTokens && a.q_heads >= 1 && a.kv_heads >= 1 && a.q_heads <= 4096 && a.kv_heads <= 4096,
              "%s: tokens=%lld q_heads=%d kv_heads=%d", who, (long long)a.tokens, a.q_heads, a.kv_heads);
  PPO_REQUIRE(a.head_dim >= 2 && a.head_dim <= PPO_QK_MAX_DIM && a.head_dim % 2 == 0, "%s: head_dim=%d (even, up to %d)", who, a.head_dim, PPO_QK_MAX_DIM);
  PPO_REQUIRE(a.rotary_dim >= 2 && a.rotary_dim <= a.head_dim && a.rotary_dim % 2 == 0, "%s: rotary_dim=%d of head_dim=%d", who, a.rotary_dim, a.head_dim);
  PPO_REQUIRE(type_ok(a.type) && (a.weight_type == a.type || a.weight_type == PPO_TYPE_F32), "%s: type=%d weight_type=%d", who, a.type, a.weight_type);
  PPO_REQUIRE(a.position_type == PPO_TOKENS_I64 || a.position_type == PPO_TOKENS_I32, "%s: position_type=%d", who, a.position_type);
  PPO_REQUIRE(a.eps >= 0.0 && a.eps < 1e30, "%s: eps=%g", who, a.eps);
  PPO_REQUIRE(a.q_weight != nullptr && a.k_weight != nullptr && a.freqs != nullptr && (a.tokens == 0 || a.positions != nullptr), "%s: null pointer", who);
  const int64_t size = type_size(a.type), wsize = type_size(a.weight_type), n = a.tokens, d = a.head_dim;
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a.q_weight) % wsize == 0 && reinterpret_cast<uintptr_t>(a.k_weight) % wsize == 0 &&
                  reinterpret_cast<uintptr_t>(a.d_q_weight) % wsize == 0 && reinterpret_cast<uintptr_t>(a.d_k_weight) % wsize == 0 &&
                  reinterpret_cast<uintptr_t>(a.freqs) % 8 == 0 &&
                  reinterpret_cast<uintptr_t>(a.positions) % (a.position_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  if (int rc = check_view(who, "q", a.q, n, a.q_heads, d, size, false)) return rc;
  if (int rc = check_view(who, "k", a.k, n, a.kv_heads, d, size, false)) return rc;
  if (int rc = check_view(who, "q_out", a.q_out, n, a.q_heads, d, size, !backward)) return rc;
  if (int rc = check_view(who, "k_out", a.k_out, n, a.kv_heads, d, size, !backward)) return rc;
  if (backward) {
    PPO_REQUIRE(a.d_q_weight != nullptr && a.d_k_weight != nullptr, "%s: null pointer", who);
    if (int rc = check_view(who, "d_q", a.d_q, n, a.q_heads, d, size, true)) return rc;
    if (int rc = check_view(who, "d_k", a.d_k, n, a.kv_heads, d, size, true)) return rc;
  }
  // apart, but for the views that a row is read from before it is written
  const int64_t qw = (a.weight_per_head != 0 ? a.q_heads : 1) * d * wsize, kw = (a.weight_per_head != 0 ? a.kv_heads : 1) * d * wsize;
  const Rows small_in[] = {vector_of(a.q_weight, qw), vector_of(a.k_weight, kw), vector_of(a.freqs, a.rotary_dim / 2 * 8),
                           vector_of(n > 0 ? a.positions : nullptr, n * (a.position_type == PPO_TOKENS_I64 ? 8 : 4))};
  const ppo_head_view* in[] = {&a.q, &a.k, backward ? &a.q_out : nullptr, backward ? &a.k_out : nullptr};
  const ppo_head_view* out[] = {backward ? &a.d_q : &a.q_out, backward ? &a.d_k : &a.k_out};
  const Rows weights_out[] = {vector_of(backward ? a.d_q_weight : nullptr, qw), vector_of(backward ? a.d_k_weight : nullptr, kw)};
  auto rows = [&](const ppo_head_view* v, int side) { return rows_of(*v, n, side == 0 ? a.q_heads : a.kv_heads, d, size); };
  for (int o = 0; o < 2; ++o) {
    const Rows x = rows(out[o], o);
    for (int i = 0; i < 4 && n > 0; ++i)
      PPO_REQUIRE(in[i] == nullptr || (i % 2 == o && same_view(*in[i], *out[o])) || !overlap(x, rows(in[i], i % 2)), "%s: an output overlaps an input", who);
    for (const Rows& y : small_in) {
      PPO_REQUIRE(n == 0 || !overlap(x, y), "%s: an output overlaps an input", who);
      PPO_REQUIRE(!overlap(weights_out[o], y), "%s: an output overlaps an input", who);
    }
    for (int i = 0; i < 4 && n > 0; ++i)
      PPO_REQUIRE(in[i] == nullptr || !overlap(weights_out[o], rows(in[i], i % 2)), "%s: an output overlaps an input", who);
    for (int w = 0; w < 2; ++w) PPO_REQUIRE(n == 0 || !overlap(x, weights_out[w]), "%s: outputs overlap", who);
  }
  PPO_REQUIRE((n == 0 || !overlap(rows(out[0], 0), rows(out[1], 1))) && !overlap(weights_out[0], weights_out[1]), "%s: outputs overlap", who);
  return PPO_OK;
}

template <class T, bool BACK>
int launch(const QkArgs& q, const Plan& p, hipStream_t st) {
  const dim3 grid(static_cast<uint32_t>(p.tiles), static_cast<uint32_t>(p.groups));
  constexpr int W = kVec<T>;
#define PPO_QK(V, U)                                                                                        \
  do {                                                                                                      \
    if constexpr (BACK) hipLaunchKernelGGL((qk_rotary_bwd_kernel<T, V, U>), grid, dim3(kThreads), 0, st, q); \
    else hipLaunchKernelGGL((qk_rotary_kernel<T, V, U>), grid, dim3(kThreads), 0, st, q);                    \
  } while (0)
  if (p.vec == W) PPO_QK(W, 1);
  else if (p.units == 1) PPO_QK(1, 1);
  else if (p.units == 2) PPO_QK(1, 2);
  else PPO_QK(1, 4);
#undef PPO_QK
  return check_launch("qk_rotary_kernel");
}

QkArgs kernel_args(const ppo_qk_rotary_args& a, const Plan& p, float* partial) {
  QkArgs q{};
  q.a = a;
  q.partial = partial;
  q.tile = p.tile;
  q.group = p.group;
  q.lanes_log2 = p.lanes_log2;
  q.inv_dim = 1.0f / static_cast<float>(a.head_dim);
  q.eps = static_cast<float>(a.eps);
  return q;
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" int ppo_qk_rotary_fwd(const ppo_qk_rotary_args* args, ppo_stream_t stream) {
  if (int rc = check("ppo_qk_rotary_fwd", args, false)) return rc;
  if (args->tokens == 0) return PPO_OK;
  const Plan p = plan_of(*args, false);
  const QkArgs q = kernel_args(*args, p, nullptr);
  int rc = PPO_OK;
  with_type(args->type, [&](auto t) { rc = launch<decltype(t), false>(q, p, static_cast<hipStream_t>(stream)); });
  return rc;
}

extern "C" size_t ppo_qk_rotary_bwd_workspace_bytes(const ppo_qk_rotary_args* args) {
  if (args == nullptr || args->tokens < 0 || args->tokens >= kMostTokens || args->head_dim < 2 || args->head_dim > PPO_QK_MAX_DIM ||
      args->q_heads < 1 || args->kv_heads < 1 || args->q_heads > 4096 || args->kv_heads > 4096)
    return 0;
  const Plan p = plan_of(*args, true);
  return 256 + static_cast<size_t>(p.rows * p.slots * args->head_dim) * sizeof(float);
}

extern "C" int ppo_qk_rotary_bwd(const ppo_qk_rotary_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream) {
  if (int rc = check("ppo_qk_rotary_bwd", args, true)) return rc;
  const size_t need = ppo_qk_rotary_bwd_workspace_bytes(args);
  PPO_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= need,
              "ppo_qk_rotary_bwd: workspace too small or not 16-byte aligned (%zu < %zu)", workspace_bytes, need);
  const Plan p = plan_of(*args, true);
  const QkArgs q = kernel_args(*args, p, static_cast<float*>(workspace));
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc = PPO_OK;
  if (args->tokens > 0) with_type(args->type, [&](auto t) { rc = launch<decltype(t), true>(q, p, st); });
  if (rc != PPO_OK) return rc;
  const dim3 grid(static_cast<uint32_t>(ceil_div(args->head_dim, kJoinWidth)), static_cast<uint32_t>(p.slots));
  const int64_t rows = args->tokens > 0 ? p.rows : 0;  // (no tokens: zeros)
  with_type(args->weight_type, [&](auto t) {
    hipLaunchKernelGGL(qk_rotary_join_kernel<decltype(t)>, grid, dim3(kJoinThreads), 0, st, q, rows);
  });
  return check_launch("qk_rotary_join_kernel");
}
