// Views [tokens, heads, elements] of the operators between a token policy's embedding and its logits: argument checks.
#pragma once

#include "elem.hpp"

namespace ppo {

// The memory of a view as rows (Rows of elem.hpp): its larger stride leads from row to row, the smaller one lies inside.
inline Rows rows_of(const ppo_head_view& v, int64_t tokens, int64_t heads, int64_t dim, int64_t size) {
  const bool by_token = heads <= 1 || (tokens > 1 && v.token_stride >= v.head_stride);
  const int64_t n = by_token ? tokens : heads, ld = by_token ? v.token_stride : v.head_stride;
  const int64_t m = by_token ? heads : tokens, inner = by_token ? v.head_stride : v.token_stride;
  const int64_t bytes = ((m > 1 ? (m - 1) * inner : 0) + dim) * size;
  return Rows{v.data, n, bytes, n > 1 ? ld * size : bytes};
}

// A view whose elements all lie at their own place: what may be written.
inline bool rows_apart(const ppo_head_view& v, int64_t tokens, int64_t heads, int64_t dim) {
  const bool by_token = heads <= 1 || (tokens > 1 && v.token_stride >= v.head_stride);
  const int64_t n = by_token ? tokens : heads, ld = by_token ? v.token_stride : v.head_stride;
  const int64_t m = by_token ? heads : tokens, inner = by_token ? v.head_stride : v.token_stride;
  return (m <= 1 || inner >= dim) && (n <= 1 || ld >= (m > 1 ? (m - 1) * inner : 0) + dim);
}

inline bool same_view(const ppo_head_view& x, const ppo_head_view& y) {
  return x.data == y.data && x.token_stride == y.token_stride && x.head_stride == y.head_stride;
}

inline int check_view(const char* who, const char* name, const ppo_head_view& v, int64_t tokens, int64_t heads, int64_t dim, int64_t size, bool written) {
  PPO_REQUIRE(tokens == 0 || v.data != nullptr, "%s: %s: null pointer", who, name);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(v.data) % size == 0, "%s: %s must be aligned to its elements", who, name);
  const int64_t most = int64_t{1} << 40;  // (so that no offset leaves 64 bits)
  PPO_REQUIRE(v.token_stride >= 0 && v.head_stride >= 0 && v.token_stride < most && v.head_stride < most, "%s: %s: strides %lld, %lld", who, name,
              (long long)v.token_stride, (long long)v.head_stride);
  PPO_REQUIRE(!written || tokens == 0 || rows_apart(v, tokens, heads, dim), "%s: rows of %s overlap", who, name);
  return PPO_OK;
}

// All waves' LDS accesses are done.  (__syncthreads() would also wait for the loads and stores on their way to and from memory, which no other wave
// of the block looks at.)
__device__ __forceinline__ void lds_barrier() { asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory"); }

}  // namespace ppo
