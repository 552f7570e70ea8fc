// One token of each of many sequences through linear attention with a decay for each head (ppo_decay_attention_step):
//   S <- f S + k v^T,   o = scale q^T S   for each query head that shares S.
//
// Bound by memory: S is read once and written once, 64 KB each way for 128 x 128.  A block takes a slice of S's columns of one row and
// head, so that few rows still fill the chip; a thread holds V neighbouring columns of up to ROWS of S's rows, all their loads in flight
// together, adds to them, stores them and sums its part of every query's product; lanes of the same columns are joined by shuffles,
// waves through LDS, in a fixed order.  1,024 rows of 8 heads of 128 x 128 (1.07 GB in and out): 209 us, the copy's rate.
#include <type_traits>

#include "views.hpp"

namespace ppo {
namespace {

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kMaxSlice = 128;
constexpr int kQueries = 4;  // query heads at a time

struct StepArgs {
  ppo_decay_step_args a;
  int32_t lanes_log2;  // lanes of a row of S in the block
  int32_t group;       // query heads of S
  float scale;
};

// V: columns of a lane.  ROWS: rows of S that a thread holds.
template <class T, int V, int ROWS>
__global__ __launch_bounds__(kThreads) void decay_step_kernel(const StepArgs q) {
  typedef float Cols __attribute__((ext_vector_type(V)));
  __shared__ float part[kQueries][kWaves][kMaxSlice];
  __shared__ float keys[PPO_DECAY_MAX_DIM], query[kQueries][PPO_DECAY_MAX_DIM];
  const ppo_decay_step_args& a = q.a;
  const int64_t row = blockIdx.x;
  const int head = blockIdx.y, lanes = 1 << q.lanes_log2, lane = threadIdx.x & (lanes - 1), first = threadIdx.x >> q.lanes_log2;
  const int apart = kThreads >> q.lanes_log2;  // a thread's rows are first + i * apart
  const int col = (blockIdx.z * lanes + lane) * V;
  // What does not hang on the slot comes first, so that the state's loads, the long ones, wait for the slot alone: a few rows take as long as their loads wait
  // for each other.
  const float log_decay = a.log_decay[head];
  int64_t slot = row;
  if (a.slots != nullptr)
    slot = a.slot_type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(a.slots)[row] : static_cast<int64_t>(static_cast<const int32_t*>(a.slots)[row]);
  const bool live = slot >= 0 && slot < a.num_slots;
  const bool fresh = a.fresh != nullptr && a.fresh[row] != 0;
  constexpr int AT_ONCE = kThreads / PPO_DECAY_MAX_DIM;  // query heads that the threads load together
  const int d = threadIdx.x % PPO_DECAY_MAX_DIM, g_of = threadIdx.x / PPO_DECAY_MAX_DIM;
  T query16[kQueries / AT_ONCE];
  auto load_queries = [&](int g0) {
#pragma unroll
    for (int i = 0; i < kQueries / AT_ONCE; ++i) {
      const int g = min(g0 + g_of + i * AT_ONCE, q.group - 1);  // (once more past the last one)
      query16[i] = (static_cast<const T*>(a.q.data) + row * a.q.token_stride + (head * q.group + g) * a.q.head_stride)[min(d, a.key_dim - 1)];
    }
  };
  auto put_queries = [&] {
#pragma unroll
    for (int i = 0; i < kQueries / AT_ONCE; ++i) query[g_of + i * AT_ONCE][d] = static_cast<float>(query16[i]);
  };
  load_queries(0);
  const T key = (static_cast<const T*>(a.k.data) + row * a.k.token_stride + head * a.k.head_stride)[min(d, a.key_dim - 1)];
  const T* values = static_cast<const T*>(a.v.data) + row * a.v.token_stride + head * a.v.head_stride;
  T v16[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v16[e] = values[min(col + e, a.value_dim - 1)];
  float* state = a.states + ((live ? slot : 0) * a.kv_heads + head) * static_cast<int64_t>(a.key_dim) * a.value_dim;
  const bool has = col < a.value_dim;
  auto out_at = [&](int g) {
    return static_cast<T*>(a.out.data) + row * a.out.token_stride + (head * q.group + g) * a.out.head_stride + col;
  };
  if (!live) {
    for (int g = first; g < q.group && has; g += apart)
#pragma unroll
      for (int e = 0; e < V; ++e) out_at(g)[e] = static_cast<T>(0.0f);
    return;
  }
  Cols s[ROWS];
  if (!fresh) {
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
      const int r = first + i * apart;
      if (r < a.key_dim && has) s[i] = *reinterpret_cast<const Cols*>(state + static_cast<int64_t>(r) * a.value_dim + col);
    }
  }
  put_queries();
  keys[d] = static_cast<float>(key);
  float v[V];
#pragma unroll
  for (int e = 0; e < V; ++e) v[e] = static_cast<float>(v16[e]);
  const float f = static_cast<float>(exp(static_cast<double>(log_decay)));
  lds_barrier();
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    const int r = first + i * apart;
    if (r < a.key_dim && has) {
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const float kv = keys[r] * v[e];
        s[i][e] = fresh ? kv : fmaf(f, s[i][e], kv);
      }
      *reinterpret_cast<Cols*>(state + static_cast<int64_t>(r) * a.value_dim + col) = s[i];
    }
  }
  for (int g0 = 0; g0 < q.group; g0 += kQueries) {
    const int count = min(kQueries, q.group - g0);
    if (g0 > 0) {
      load_queries(g0);
      lds_barrier();
      put_queries();
      lds_barrier();
    }
    auto sums = [&](auto at_once, int g) {  // (together, so that their shuffles do not wait for each other)
      constexpr int N = at_once;
      float o[N][V] = {};
#pragma unroll
      for (int i = 0; i < ROWS; ++i) {
        const int r = first + i * apart;
        if (r < a.key_dim && has)
#pragma unroll
          for (int h = 0; h < N; ++h)
#pragma unroll
            for (int e = 0; e < V; ++e) o[h][e] = fmaf(query[g + h][r], s[i][e], o[h][e]);
      }
      for (int w = lanes; w < kWave; w <<= 1)
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
          for (int e = 0; e < V; ++e) o[h][e] += __shfl_xor(o[h][e], w, kWave);
      if (threadIdx.x % kWave < static_cast<uint32_t>(lanes))
#pragma unroll
        for (int h = 0; h < N; ++h)
#pragma unroll
          for (int e = 0; e < V; ++e) part[g + h][threadIdx.x / kWave][lane * V + e] = o[h][e];
    };
    if (count == kQueries) sums(std::integral_constant<int, kQueries>{}, 0);
    else
      for (int g = 0; g < count; ++g) sums(std::integral_constant<int, 1>{}, g);
    lds_barrier();
    for (int g = first; g < count && has; g += apart)
#pragma unroll
      for (int e = 0; e < V; ++e) {
        const int c = lane * V + e;
        out_at(g0 + g)[e] = static_cast<T>(q.scale * ((part[g][0][c] + part[g][1][c]) + (part[g][2][c] + part[g][3][c])));
      }
  }
}

template <class T>
void launch(const StepArgs& q, bool fours, hipStream_t st) {
  const ppo_decay_step_args& a = q.a;
  const int v = fours ? 4 : 1, lanes = 1 << q.lanes_log2;
  const dim3 grid(static_cast<uint32_t>(a.rows), static_cast<uint32_t>(a.kv_heads), static_cast<uint32_t>(ceil_div(a.value_dim, lanes * v)));
  const int rows = static_cast<int>(ceil_div(a.key_dim, kThreads >> q.lanes_log2));
#define PPO_STEP(V, ROWS) hipLaunchKernelGGL((decay_step_kernel<T, V, ROWS>), grid, dim3(kThreads), 0, st, q)
  if (fours) {
    if (rows <= 4) PPO_STEP(4, 4);
    else if (rows <= 8) PPO_STEP(4, 8);
    else PPO_STEP(4, 16);
  } else {
    if (rows <= 4) PPO_STEP(1, 4);
    else if (rows <= 16) PPO_STEP(1, 16);
    else PPO_STEP(1, 32);
  }
#undef PPO_STEP
}

int check(const ppo_decay_step_args& a) {
  const char* who = "ppo_decay_attention_step";
  PPO_REQUIRE(a.rows >= 0 && a.rows < (int64_t{1} << 24) && a.num_slots >= 0 && a.num_slots < INT32_MAX, "%s: rows=%lld num_slots=%lld", who, (long long)a.rows,
              (long long)a.num_slots);
  PPO_REQUIRE(a.q_heads >= 1 && a.kv_heads >= 1 && a.q_heads <= 65535 && a.q_heads % a.kv_heads == 0, "%s: q_heads=%d kv_heads=%d", who, a.q_heads, a.kv_heads);
  PPO_REQUIRE(a.key_dim >= 1 && a.key_dim <= PPO_DECAY_MAX_DIM && a.value_dim >= 1 && a.value_dim <= PPO_DECAY_MAX_DIM,
              "%s: key_dim=%d value_dim=%d (1 to %d)", who, a.key_dim, a.value_dim, PPO_DECAY_MAX_DIM);
  PPO_REQUIRE(type_ok(a.type), "%s: type=%d", who, a.type);
  PPO_REQUIRE(a.slot_type == PPO_TOKENS_I64 || a.slot_type == PPO_TOKENS_I32, "%s: slot_type=%d", who, a.slot_type);
  PPO_REQUIRE(a.scale > -1e30 && a.scale < 1e30, "%s: scale=%g", who, a.scale);
  PPO_REQUIRE(a.slots != nullptr || a.rows <= a.num_slots, "%s: %lld rows for %lld states", who, (long long)a.rows, (long long)a.num_slots);
  PPO_REQUIRE(a.log_decay != nullptr && (a.states != nullptr || a.num_slots == 0), "%s: null pointer", who);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a.log_decay) % 4 == 0 && reinterpret_cast<uintptr_t>(a.states) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(a.slots) % (a.slot_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  const int64_t n = a.rows, size = type_size(a.type), dk = a.key_dim, dv = a.value_dim;
  if (int rc = check_view(who, "q", a.q, n, a.q_heads, dk, size, false)) return rc;
  if (int rc = check_view(who, "k", a.k, n, a.kv_heads, dk, size, false)) return rc;
  if (int rc = check_view(who, "v", a.v, n, a.kv_heads, dv, size, false)) return rc;
  if (int rc = check_view(who, "out", a.out, n, a.q_heads, dv, size, true)) return rc;
  if (n == 0) return PPO_OK;
  const Rows states = vector_of(a.states, a.num_slots * a.kv_heads * dk * dv * 4), out = rows_of(a.out, n, a.q_heads, dv, size);
  const Rows in[] = {rows_of(a.q, n, a.q_heads, dk, size), rows_of(a.k, n, a.kv_heads, dk, size), rows_of(a.v, n, a.kv_heads, dv, size),
                     vector_of(a.log_decay, a.kv_heads * 4), vector_of(a.slots, n * (a.slot_type == PPO_TOKENS_I64 ? 8 : 4)), vector_of(a.fresh, n)};
  for (const Rows& x : in) PPO_REQUIRE(!overlap(out, x) && !overlap(states, x), "%s: an output overlaps an input", who);
  PPO_REQUIRE(!overlap(out, states), "%s: outputs overlap", who);
  return PPO_OK;
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" int ppo_decay_attention_step(const ppo_decay_step_args* args, ppo_stream_t stream) {
  PPO_REQUIRE(args != nullptr, "ppo_decay_attention_step: null arguments");
  if (int rc = check(*args)) return rc;
  const ppo_decay_step_args& a = *args;
  if (a.rows == 0) return PPO_OK;
  StepArgs q{};
  q.a = a;
  q.group = a.q_heads / a.kv_heads;
  q.scale = static_cast<float>(a.scale);
  const bool fours = a.value_dim % 4 == 0 && reinterpret_cast<uintptr_t>(a.states) % 16 == 0;
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  // as many columns as a block takes, unless that leaves the chip idle (8 rows of 4 heads: 6.5 us with 128 columns a block, 4.5 with 32; 256 rows of 8 heads:
  // 42.8 and 44.5)
  const int v = fours ? 4 : 1;
  q.lanes_log2 = 0;
  while ((1 << q.lanes_log2) * v < a.value_dim && q.lanes_log2 < (fours ? 5 : 6)) ++q.lanes_log2;
  while (q.lanes_log2 > 3 && a.rows * a.kv_heads * ceil_div(a.value_dim, (1 << q.lanes_log2) * v) < 2 * cus) --q.lanes_log2;
  with_type(a.type, [&](auto t) { launch<decltype(t)>(q, fours, static_cast<hipStream_t>(stream)); });
  return check_launch("decay_step_kernel");
}
