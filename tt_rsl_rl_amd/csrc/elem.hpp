// Element types of the token operators (embedding.hip, token_loss.hip, adamw.hip): fp32, bf16 and fp16 in memory, fp32 in
// registers.  A rounding to 16 bits is to nearest even (gfx950's converts), once, at a store.
#pragma once

#include "common.hpp"

namespace ppo {

constexpr int kTypes = 3;
__host__ __device__ constexpr int type_size(int type) { return type == PPO_TYPE_F32 ? 4 : 2; }
inline bool type_ok(int type) { return type >= 0 && type < kTypes; }

template <class T>
constexpr int kVec = 16 / static_cast<int>(sizeof(T));  // elements of a 16-byte piece

// A 16-byte piece that need not lie on a 16-byte boundary (rows of an odd width): gfx950 loads and stores it in one
// instruction all the same, at one more cache line per wave.
template <class T>
struct Piece {
  typedef T type __attribute__((ext_vector_type(16 / sizeof(T)), aligned(sizeof(T))));
};

// A piece as it lies in memory, four registers whatever the type, for values that are kept and converted where they are used.
// (An array: element reads of a vector through a reference are miscompiled, all of them to the first element.)
struct RawPiece {
  uint32_t w[4];
};

template <class T>
__device__ __forceinline__ float element(const RawPiece& r, int e) {
  if constexpr (sizeof(T) == 4) {
    return __builtin_bit_cast(float, r.w[e]);
  } else {
    const uint32_t w = r.w[e / 2];
    if constexpr (__is_same(T, __bf16)) return __builtin_bit_cast(float, e % 2 != 0 ? w & 0xffff0000u : w << 16);
    else return static_cast<float>(__builtin_bit_cast(T, static_cast<uint16_t>(e % 2 != 0 ? w >> 16 : w)));
  }
}

// Makes element e -inf.
template <class T>
__device__ __forceinline__ void make_neg_inf(RawPiece& r, int e) {
  if constexpr (sizeof(T) == 4) {
    r.w[e] = 0xff800000u;
  } else {
    const uint32_t bits = __is_same(T, __bf16) ? 0xff80u : 0xfc00u;
    r.w[e / 2] = e % 2 != 0 ? (r.w[e / 2] & 0xffffu) | bits << 16 : (r.w[e / 2] & 0xffff0000u) | bits;
  }
}

// The compiler forgets what it knows of the piece, once `done` is computed: otherwise it keeps the converted values of one
// pass for the next, or puts the pass off, at two or more registers for each of the piece's.
__device__ __forceinline__ void forget(RawPiece& r, float& done) { asm volatile("" : "+v"(r.w[0]), "+v"(r.w[1]), "+v"(r.w[2]), "+v"(r.w[3]), "+v"(done)); }
__device__ __forceinline__ void forget(int& x) { asm volatile("" : "+v"(x)); }

// A loaded value that has to have arrived here: what follows may overwrite where it came from.
__device__ __forceinline__ void arrived(float& x) { asm volatile("" : "+v"(x)); }

// STREAM: past the caches.  For calls that touch more than the last-level cache holds: nothing of it will still be there when it is
// next used, and what is written through the cache leaves dirty lines in the way of what is read meanwhile.  Both sides measured
// (us, through the caches -> past them): embedding gradient of 256 MiB summands into a 256 MiB table 187 -> 141, with a reader of
// the table behind it 314 -> 269 (512 MiB), but 94.4 -> 98.7 (128 MiB); loss of 250 MiB logits 111.8 -> 106.4; AdamW touching 341 MiB
// 124.1 -> 119.5, 171 MiB 60.6 -> 66.0.
constexpr int64_t kCacheBytes = int64_t{1} << 28;

template <bool STREAM = false, class T>
__device__ __forceinline__ typename Piece<T>::type load_piece(const T* p) {
  const auto* q = reinterpret_cast<const typename Piece<T>::type*>(p);
  if constexpr (STREAM) return __builtin_nontemporal_load(q);
  else return *q;
}

template <bool STREAM = false, class T>
__device__ __forceinline__ RawPiece load_raw(const T* p) {
  return __builtin_bit_cast(RawPiece, load_piece<STREAM>(p));
}

template <bool STREAM = false, class T>
__device__ __forceinline__ void store_piece(T* p, const float (&x)[kVec<T>]) {
  typename Piece<T>::type v;
#pragma unroll
  for (int i = 0; i < kVec<T>; ++i) v[i] = static_cast<T>(x[i]);
  auto* q = reinterpret_cast<typename Piece<T>::type*>(p);
  if constexpr (STREAM) __builtin_nontemporal_store(v, q);
  else *q = v;
}

// Tokens are int64 or int32; anything outside [0, vocab) is no token (-1).
__device__ __forceinline__ int64_t token_at(const void* tokens, int type, int64_t i, int64_t vocab) {
  const int64_t t = type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(tokens)[i]
                                           : static_cast<int64_t>(static_cast<const int32_t*>(tokens)[i]);
  return t >= 0 && t < vocab ? t : -1;
}

// Memory that a call reads and memory that it writes: one block may write what another has yet to read, so an output may not lie
// on an input unless the header says so.  Rows of a matrix, in bytes.
struct Rows {
  const void* at;
  int64_t rows, bytes, ld;
};
inline bool overlap(const Rows& x, const Rows& y) {
  if (x.at == nullptr || y.at == nullptr || x.rows <= 0 || y.rows <= 0) return false;
  const int64_t a = static_cast<int64_t>(reinterpret_cast<uintptr_t>(x.at)), b = static_cast<int64_t>(reinterpret_cast<uintptr_t>(y.at));
  if (a + (x.rows - 1) * x.ld + x.bytes <= b || b + (y.rows - 1) * y.ld + y.bytes <= a) return false;
  if (x.ld != y.ld) return true;
  const int64_t apart = ((b - a) % x.ld + x.ld) % x.ld;  // columns of one matrix may lie side by side
  return apart < x.bytes || apart + y.bytes > x.ld;
}
inline Rows vector_of(const void* p, int64_t bytes) { return Rows{p, 1, bytes, bytes}; }

// f(T()) for the element type of `type`.
template <class F>
void with_type(int type, F&& f) {
  if (type == PPO_TYPE_F32) f(float());
  else if (type == PPO_TYPE_BF16) f(static_cast<__bf16>(0.0f));
  else f(static_cast<_Float16>(0.0f));
}

}  // namespace ppo
