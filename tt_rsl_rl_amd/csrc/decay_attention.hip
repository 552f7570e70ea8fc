// Linear attention whose past fades by a factor for each head: chunks on the matrix cores (ppo_decay_attention_fwd, _bwd) and single
// tokens (ppo_decay_attention_step).
//
// All four results are one sum, with tokens in order or in reverse (positions u in the order that is walked, w = 1 or 0):
//   out_i = x sum_{j <= i} f^(i-j) (a_i . b_j) c_j  +  y f^(i+w) a_i S,      S <- f^n S + z sum_j f^(n-w-j) b_j c_j^T
//   o:   a = q, b = k, c = v,      in order,    w = 1, x = y = scale, z = 1     S [key, value]
//   d_q: a = d_o, b = v, c = k,    in order,    w = 1, x = y = scale, z = 1     S [value, key]
//   d_v: a = k, b = q, c = d_o,    in reverse,  w = 0, x = z = scale, y = 1     R [key, value]   (b and c over the heads that share k)
//   d_k: a = v, b = d_o, c = q,    in reverse,  w = 0, x = z = scale, y = 1     R [value, key]
// (in reverse what is handed on is f R, since the gradient of the last state enters undecayed).
//
// A block walks the chunks of a segment of tokens for one head of b and c (GA heads of a read them) or of a (GB heads of b and c are
// summed).  S stays in its waves' accumulators, each wave owning columns of c; the accumulator layout (column lane % 16, rows
// 4 (lane / 16) + 0..3) is that of an operand whose sum runs over those rows, in fours, so neither S nor the chunk's matrix passes
// through LDS on its way into the next product.  Each wave makes the chunk's whole matrix for itself: that costs less than the
// barrier and the LDS traffic of sharing it.  Operands that are sums themselves (S, the matrix, weighted c) go into bf16 products as 2, 2
// and 3 parts of 8 bits each: S and the matrix then add 2^-17 to outputs that are rounded to 2^-9 anyway, and a state, which is
// fp32, keeps 2^-24.  fp16 goes through the fp32 products: a state may leave fp16's range, and two bf16 parts of it would need
// two of q as well.
// With few heads the sequence is cut into segments: a first pass makes each segment's own state, a scan carries them on, and the second pass
// starts every segment from the state before it.
//
// Sequences lie one after another at any offset.  Chunks are cut at multiples of the chunk alone, and the matrix is masked where
// sequences differ; where states come in or go out, chunks are cut at the sequences' ends too.
// A token whose b or c is not finite would reach, as 0 * inf, tokens that do not see it: its row is taken as zeros, and NaN put into
// what does see it.
#include <type_traits>

#include "views.hpp"

namespace ppo {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kThreads = 256;
constexpr int kWaves = kThreads / kWave;
constexpr int kInfoThreads = 256;
constexpr int kScanThreads = 256;

// The matrix cores' operand types.  A step sums over K elements: QUADS groups of four for each of a wave's four lane groups g, group h
// being elements 16 h + 4 g + 0..3 of the step.
template <class M>
struct Math;
template <>
struct Math<__bf16> {
  static constexpr int K = 32, QUADS = 2, CHUNK = 64, PARTS2 = 2, PARTS3 = 3;
  typedef bf16x8 Frag;
  typedef bf16x4 Quad;
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, const f32x4& c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b, c, 0, 0, 0);
  }
};
template <>
struct Math<float> {
  static constexpr int K = 16, QUADS = 1, CHUNK = 32, PARTS2 = 1, PARTS3 = 1;
  typedef f32x4 Frag;
  typedef f32x4 Quad;
  static __device__ __forceinline__ f32x4 mma(const Frag& a, const Frag& b, f32x4 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
};

// An operand from LDS: row[base + 16 h + 4 g ..], g the lane's group.
template <class M>
__device__ __forceinline__ typename Math<M>::Frag load_frag(const M* row, int base, int g) {
  typedef typename Math<M>::Quad Quad;
  if constexpr (Math<M>::QUADS == 1) {
    return *reinterpret_cast<const Quad*>(row + base + 4 * g);
  } else {
    const Quad u = *reinterpret_cast<const Quad*>(row + base + 4 * g), v = *reinterpret_cast<const Quad*>(row + base + 16 + 4 * g);
    return __builtin_shufflevector(u, v, 0, 1, 2, 3, 4, 5, 6, 7);
  }
}

// Values of a step as NP operands whose sum they are, to 8 bits each (bf16), or as they are (fp32).
template <class M, int NP>
__device__ __forceinline__ void split(float (&x)[4 * Math<M>::QUADS], typename Math<M>::Frag (&out)[NP]) {
#pragma unroll
  for (int p = 0; p < NP; ++p)
#pragma unroll
    for (int i = 0; i < 4 * Math<M>::QUADS; ++i) {
      const M part = static_cast<M>(x[i]);
      out[p][i] = part;
      if (p + 1 < NP) x[i] -= static_cast<float>(part);
    }
}

struct Span {
  int32_t start, end, seq;  // seq -1: the token belongs to no sequence
};

struct MixArgs {
  ppo_head_view a, b, c, out;
  const float* log_decay;
  const Span* spans;    // of each token; NULL: one sequence
  const float* s_in;    // [sequences][heads][elements], element (b's dim i, c's dim j) at i * si + j * sj
  float* s_out;
  float* carry;         // [segments - 1][heads][db][dc]: the state that leaves a segment, then what enters the next
  int64_t si, sj, state_size;
  int32_t tokens, segment, segments;
  int32_t heads, ga, gb;  // heads of b, c and S times gb; of a per head
  int32_t db, dc;
  int32_t reverse, w, cut;  // cut: chunks end with their sequence
  float x, y, z;
};

__device__ __forceinline__ Span span_of(const MixArgs& q, int token) {
  return q.spans == nullptr ? Span{0, q.tokens, 0} : q.spans[token];
}

// One thread a token: the sequence that it lies in.
__global__ __launch_bounds__(kInfoThreads) void decay_spans_kernel(const void* cu, int cu_type, int sequences, int tokens, Span* spans) {
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kInfoThreads + threadIdx.x;
  if (t >= tokens) return;
  auto at = [&](int i) {
    return cu_type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(cu)[i] : static_cast<int64_t>(static_cast<const int32_t*>(cu)[i]);
  };
  int lo = 0, hi = sequences + 1;  // the first entry above t
  while (lo < hi) {
    const int mid = (lo + hi) / 2;
    if (at(mid) > t) hi = mid;
    else lo = mid + 1;
  }
  Span s{static_cast<int32_t>(t), static_cast<int32_t>(t) + 1, -1};
  if (lo >= 1 && lo <= sequences) {
    const int64_t from = max(at(lo - 1), static_cast<int64_t>(0)), to = min(at(lo), static_cast<int64_t>(tokens));
    if (from <= t && to > t) s = Span{static_cast<int32_t>(from), static_cast<int32_t>(to), lo - 1};
  }
  spans[t] = s;
}

// A sequence without tokens hands its state on.
__global__ __launch_bounds__(256) void decay_empty_kernel(const void* cu, int cu_type, int tokens, const float* from, float* to, int64_t size) {
  const int64_t b = blockIdx.x;
  auto at = [&](int64_t i) {
    const int64_t v = cu_type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(cu)[i] : static_cast<int64_t>(static_cast<const int32_t*>(cu)[i]);
    return min(max(v, static_cast<int64_t>(0)), static_cast<int64_t>(tokens));
  };
  const bool empty = cu == nullptr ? tokens == 0 : at(b + 1) <= at(b);
  if (!empty) return;
  for (int64_t i = threadIdx.x; i < size; i += 256) to[b * size + i] = from == nullptr ? 0.0f : from[b * size + i];
}

// carry[s] holds what segment s makes of nothing; afterwards what enters segment s + 1.
__global__ __launch_bounds__(kScanThreads) void decay_scan_kernel(const MixArgs q) {
  const int64_t size = static_cast<int64_t>(q.db) * q.dc, i = static_cast<int64_t>(blockIdx.x) * kScanThreads + threadIdx.x;
  const int h = blockIdx.y;
  if (i >= size) return;
  const float ld = q.log_decay[h], whole = static_cast<float>(exp(static_cast<double>(ld) * q.segment));
  float* at = q.carry + h * size + i;
  const int64_t step = size * q.heads;
  float s = 0.0f;
  constexpr int AHEAD = 8;
  for (int g = 0; g < q.segments - 1; g += AHEAD) {
    float own[AHEAD];
    bool kept[AHEAD];
#pragma unroll
    for (int e = 0; e < AHEAD; ++e) {
      const int seg = min(g + e, q.segments - 2);
      own[e] = at[seg * step];
      const int u = (seg + 1) * q.segment - 1;  // the segment's last position; its sequence came from before the segment?
      const Span s0 = span_of(q, q.reverse ? q.tokens - 1 - u : u);
      kept[e] = (q.reverse ? q.tokens - s0.end : s0.start) < seg * q.segment;
    }
#pragma unroll
    for (int e = 0; e < AHEAD; ++e)
      if (g + e < q.segments - 1) {
        s = kept[e] ? fmaf(whole, s, own[e]) : own[e];
        at[(g + e) * step] = s;
      }
  }
}

// Four tokens' pieces of 16 bytes of one view, as they lie in memory; zeros past the view's rows and columns.
template <class T>
struct Unit {
  RawPiece r[4];
};

template <class T>
__device__ __forceinline__ RawPiece load_columns(const T* row, int col, int dim) {
  constexpr int V = kVec<T>;
  if (col + V <= dim) return load_raw(row + col);
  RawPiece r{};
  for (int e = 0; e < V; ++e)
    if (col + e < dim) {
      if constexpr (sizeof(T) == 4) r.w[e] = __builtin_bit_cast(uint32_t, row[col + e]);
      else r.w[e / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, row[col + e])) << (e % 2 * 16);
    }
  return r;
}

// Whether any of the piece's values is not finite.
template <class T>
__device__ __forceinline__ uint32_t not_finite(const RawPiece& r) {
  uint32_t any = 0;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) any |= ((r.w[i] & 0x7fffffffu) + 0x00800000u) & 0x80000000u;
    else if constexpr (__is_same(T, __bf16)) any |= ((r.w[i] & 0x7fff7fffu) + 0x00800080u) & 0x80008000u;
    else any |= ((r.w[i] & 0x7fff7fffu) + 0x04000400u) & 0x80008000u;
  }
  return any;
}

template <class M>
constexpr int natural_stride(int dim) { return dim + (sizeof(M) == 2 ? 8 : 4); }
template <class M>
constexpr int turned_stride() { return Math<M>::CHUNK + 4; }

// T: the views' type, M: the products', DBT: tiles of 16 of b's dims, NT: tiles of 16 of c's dims a wave owns, STATE_ONLY: the first pass over
// segments, which makes their own states.
template <class T, class M, int DBT, int NT, bool STATE_ONLY>
__global__ __launch_bounds__(kThreads, sizeof(M) == 2 ? 2 : 1) void decay_mix_kernel(const MixArgs q) {
  typedef Math<M> X;
  typedef typename X::Frag Frag;
  constexpr int C = X::CHUNK, K = X::K, Q = X::QUADS, DB = DBT * 16, DC = kWaves * NT * 16, IT = C / 16, V = kVec<T>;
  constexpr int SN = natural_stride<M>(DB), ST = turned_stride<M>();
  __shared__ __align__(16) M a_rows[STATE_ONLY ? 8 : C * SN];
  __shared__ __align__(16) M b_rows[STATE_ONLY ? 8 : C * SN];
  __shared__ __align__(16) M b_turned[DB * ST];
  __shared__ __align__(16) M c_turned[DC * ST];
  __shared__ float fades[C + 1];
  __shared__ int first[C + 1], last[C + 1], seqs[C];
  __shared__ uint32_t bad_any;
  __shared__ uint32_t bad[(C + 31) / 32];

  const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave, col = lane % 16, g = lane / 16;
  const int head = blockIdx.y, seg = blockIdx.x;
  const int dc0 = wave * NT * 16;
  const bool works = dc0 < q.dc;
  const int seg_begin = seg * q.segment, seg_end = min(seg_begin + q.segment, q.tokens);
  const double ld = static_cast<double>(q.log_decay[head]);
  if (threadIdx.x <= C) fades[threadIdx.x] = threadIdx.x == 0 ? 1.0f : static_cast<float>(exp(ld * threadIdx.x));
  if (threadIdx.x == 0) bad_any = 0;

  f32x4 S[DBT][NT];
  auto each_state = [&](auto&& f) {
#pragma unroll
    for (int mb = 0; mb < DBT; ++mb)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[mb][nt][r] = f(S[mb][nt][r], 16 * mb + 4 * g + r, dc0 + 16 * nt + col);
  };
  each_state([](float, int, int) { return 0.0f; });
  bool fresh = true;  // S is zeros

  for (int c0 = seg_begin; c0 < seg_end; c0 += C) {
    const int cn = min(C, seg_end - c0);
    __syncthreads();
    if (threadIdx.x < static_cast<uint32_t>(cn)) {
      const int u = c0 + threadIdx.x;
      const Span s = span_of(q, q.reverse ? q.tokens - 1 - u : u);
      first[threadIdx.x] = q.reverse ? q.tokens - s.end : s.start;
      last[threadIdx.x] = q.reverse ? q.tokens - s.start : s.end;
      seqs[threadIdx.x] = s.seq;
    }
    __syncthreads();
    if (!STATE_ONLY && c0 == seg_begin && first[0] < c0) {  // goes on from the segment before
      const float* from = q.carry + (static_cast<int64_t>(seg - 1) * q.heads + head) * q.db * q.dc;
      each_state([&](float, int i, int j) { return works && i < q.db && j < q.dc ? from[static_cast<int64_t>(i) * q.dc + j] : 0.0f; });
      fresh = false;
    }
    for (int p = 0; p < cn;) {
      const int begin = c0 + p, seq = __builtin_amdgcn_readfirstlane(seqs[p]), first0 = __builtin_amdgcn_readfirstlane(first[p]);
      const int n = __builtin_amdgcn_readfirstlane(q.cut ? min(cn - p, last[p] - begin) : cn - p);
      if (first0 == begin) {  // a sequence begins
        fresh = q.s_in == nullptr || seq < 0;
        const float* from = q.s_in + (static_cast<int64_t>(seq) * q.heads + head) * q.state_size;
        each_state([&](float, int i, int j) { return !fresh && works && i < q.db && j < q.dc ? from[i * q.si + j * q.sj] : 0.0f; });
      }
      const int first_last = __builtin_amdgcn_readfirstlane(first[p + n - 1]);  // where the sequence of the last token begins
      f32x4 acc[IT][NT];
      for (int ab = 0; ab < q.ga * q.gb; ++ab) {
        const int ha = q.ga > 1 ? head * q.ga + ab : head, hb = q.gb > 1 ? head * q.gb + ab : head;
        const bool new_b = q.gb > 1 || ab == 0, new_a = !STATE_ONLY && (q.ga > 1 || ab == 0);
        __syncthreads();
        // rows into LDS: units of four tokens by 16 bytes of a head
        auto stage = [&](const ppo_head_view& v, int h, int dim, int padded, M* rows, M* turned, bool check) {
          const int pieces = padded / V;
          for (int i = threadIdx.x; i < pieces * (C / 4); i += kThreads) {
            const int j4 = i / pieces * 4, d = i % pieces * V;
            RawPiece r[4];
            uint32_t any[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              const int j = j4 + k;
              r[k] = RawPiece{};
              if (j < n && seqs[p + j] >= 0) {
                const int u = begin + j, t = q.reverse ? q.tokens - 1 - u : u;
                r[k] = load_columns(static_cast<const T*>(v.data) + t * v.token_stride + h * v.head_stride, d, dim);
              }
            }
            if (check) {
#pragma unroll
              for (int k = 0; k < 4; ++k) any[k] = not_finite<T>(r[k]);
              if ((any[0] | any[1] | any[2] | any[3]) != 0) {
                for (int k = 0; k < 4; ++k)
                  if (any[k] != 0) atomicOr(&bad[(j4 + k) / 32], 1u << ((j4 + k) % 32));
                bad_any = 1;
              }
            }
            if (rows != nullptr)
#pragma unroll
              for (int k = 0; k < 4; ++k) {
                typedef M Row __attribute__((ext_vector_type(V)));
                Row x;
#pragma unroll
                for (int e = 0; e < V; ++e) x[e] = static_cast<M>(element<T>(r[k], e));
                typedef M Part __attribute__((ext_vector_type(16 / sizeof(M))));
                constexpr int PV = 16 / static_cast<int>(sizeof(M));
#pragma unroll
                for (int e = 0; e < V; e += PV) {
                  Part y;
#pragma unroll
                  for (int f = 0; f < PV; ++f) y[f] = x[e + f];
                  *reinterpret_cast<Part*>(rows + (j4 + k) * SN + d + e) = y;
                }
              }
            if (turned != nullptr)
#pragma unroll
              for (int e = 0; e < V; ++e) {
                typename X::Quad x;
#pragma unroll
                for (int k = 0; k < 4; ++k) x[k] = static_cast<M>(element<T>(r[k], e));
                *reinterpret_cast<typename X::Quad*>(turned + (d + e) * ST + j4) = x;
              }
          }
        };
        if (new_b && threadIdx.x < (C + 31) / 32) bad[threadIdx.x] = 0;
        if (new_b) __syncthreads();
        if (new_a) stage(q.a, ha, q.db, DB, a_rows, nullptr, false);
        if (new_b) {
          stage(q.b, hb, q.db, DB, STATE_ONLY ? nullptr : b_rows, b_turned, true);
          stage(q.c, hb, q.dc, DC, nullptr, c_turned, true);
        }
        __syncthreads();
        const bool poisoned = __builtin_amdgcn_readfirstlane(bad_any) != 0;
        if (poisoned) {  // zeros where a token is not finite; rare, so one token after another
          for (int j = 0; j < n; ++j)
            if (bad[j / 32] >> (j % 32) & 1) {
              for (int d = threadIdx.x; d < DB; d += kThreads) {
                if (!STATE_ONLY) b_rows[j * SN + d] = static_cast<M>(0.0f);
                b_turned[d * ST + j] = static_cast<M>(0.0f);
              }
              for (int d = threadIdx.x; d < DC; d += kThreads) c_turned[d * ST + j] = static_cast<M>(0.0f);
            }
          __syncthreads();
        }
        // ---- what lies before the piece ----
        if (!STATE_ONLY && (ab == 0 || q.ga > 1)) {
#pragma unroll
          for (int it = 0; it < IT; ++it)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) acc[it][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
          if (works && !fresh) {
#pragma unroll
            for (int ks = 0; ks < DB / K; ++ks) {
              Frag s[NT][X::PARTS2];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float v[4 * Q];
#pragma unroll
                for (int i = 0; i < 4 * Q; ++i) v[i] = S[ks * Q + i / 4][nt][i % 4];
                split<M, X::PARTS2>(v, s[nt]);
              }
#pragma unroll
              for (int it = 0; it < IT; ++it) {
                const Frag a = load_frag<M>(a_rows + (16 * it + col) * SN, K * ks, g);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int k = 0; k < X::PARTS2; ++k) acc[it][nt] = X::mma(s[nt][k], a, acc[it][nt]);
              }
            }
#pragma unroll
            for (int it = 0; it < IT; ++it) {
              const int i = 16 * it + col;
              const bool sees = i < n && first[p + min(i, n - 1)] == first0;
              const float f = q.y * fades[min(i + q.w, C)];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int r = 0; r < 4; ++r) acc[it][nt][r] = sees ? acc[it][nt][r] * f : 0.0f;
            }
          }
        }
        // c's columns that the wave owns, as operands
        Frag c[NT][C / K];
        if (works)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int ks = 0; ks < C / K; ++ks) c[nt][ks] = load_frag<M>(c_turned + (dc0 + 16 * nt + col) * ST, K * ks, g);
        // ---- the piece's tokens among each other ----
        if (!STATE_ONLY && works) {
          const bool one = first_last == first0 && seq >= 0;  // one sequence
#pragma unroll
          for (int it = 0; it < IT; ++it) {
            if (16 * it >= n) break;
            Frag a[DB / K];
#pragma unroll
            for (int ks = 0; ks < DB / K; ++ks) a[ks] = load_frag<M>(a_rows + (16 * it + col) * SN, K * ks, g);
            const int i = 16 * it + col, first_i = first[p + min(i, n - 1)];
#pragma unroll
            for (int kj = 0; kj < C / K; ++kj) {
              if (kj * Q > it) continue;
              float v[4 * Q];
#pragma unroll
              for (int h = 0; h < Q; ++h) {
                const int jt = kj * Q + h;
                f32x4 m{0.0f, 0.0f, 0.0f, 0.0f};
                if (jt <= it) {
#pragma unroll
                  for (int ks = 0; ks < DB / K; ++ks) m = X::mma(load_frag<M>(b_rows + (16 * jt + col) * SN, K * ks, g), a[ks], m);
#pragma unroll
                  for (int r = 0; r < 4; ++r) {
                    const int j = 16 * jt + 4 * g + r;
                    const bool sees = j <= i && i < n && (one || first[p + min(j, n - 1)] == first_i);
                    m[r] = sees ? m[r] * (q.x * fades[max(i - j, 0)]) : 0.0f;
                  }
                }
#pragma unroll
                for (int r = 0; r < 4; ++r) v[4 * h + r] = m[r];
              }
              Frag part[X::PARTS2];
              split<M, X::PARTS2>(v, part);
#pragma unroll
              for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                for (int k = 0; k < X::PARTS2; ++k) acc[it][nt] = X::mma(c[nt][kj], part[k], acc[it][nt]);
            }
            if (poisoned)
              for (int j = 0; j <= min(i, n - 1); ++j)
                if ((bad[j / 32] >> (j % 32) & 1) && first[p + j] == first_i)
#pragma unroll
                  for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int r = 0; r < 4; ++r) acc[it][nt][r] = __builtin_nanf("");
          }
        }
        // ---- the outputs ----
        if (!STATE_ONLY && works && (q.ga > 1 || ab == q.gb - 1)) {
#pragma unroll
          for (int it = 0; it < IT; ++it) {
            const int i = 16 * it + col;
            if (i < n && seqs[p + min(i, n - 1)] >= 0) {
              const int u = begin + i, t = q.reverse ? q.tokens - 1 - u : u;
              T* row = static_cast<T*>(q.out.data) + t * q.out.token_stride + ha * q.out.head_stride;
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                const int d = dc0 + 16 * nt + 4 * g;
                if (d + 4 <= q.dc) {
                  typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
                  Four o;
#pragma unroll
                  for (int r = 0; r < 4; ++r) o[r] = static_cast<T>(acc[it][nt][r]);
                  *reinterpret_cast<Four*>(row + d) = o;
                } else {
#pragma unroll
                  for (int r = 0; r < 4; ++r)
                    if (d + r < q.dc) row[d + r] = static_cast<T>(acc[it][nt][r]);
                }
              }
            }
          }
        }
        // ---- the state ----
        if (ab >= q.ga - 1) {
          const bool kept = first_last == first0;
          if (ab == q.ga - 1) {
            const float f = fades[n];
            each_state([&](float s, int, int) { return kept ? s * f : 0.0f; });
          }
          if (works) {
#pragma unroll
            for (int kj = 0; kj < C / K; ++kj) {
              float w[4 * Q];
#pragma unroll
              for (int i = 0; i < 4 * Q; ++i) {
                const int j = K * kj + 16 * (i / 4) + 4 * g + i % 4;
                w[i] = j < n && first[p + min(j, n - 1)] == first_last ? q.z * fades[max(n - q.w - j, 0)] : 0.0f;
              }
              Frag weighted[NT][X::PARTS3];
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) {
                float v[4 * Q];
#pragma unroll
                for (int i = 0; i < 4 * Q; ++i) v[i] = w[i] * static_cast<float>(c[nt][kj][i]);
                split<M, X::PARTS3>(v, weighted[nt]);
              }
#pragma unroll
              for (int mb = 0; mb < DBT; ++mb) {
                const Frag b = load_frag<M>(b_turned + (16 * mb + col) * ST, K * kj, g);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                  for (int k = 0; k < X::PARTS3; ++k) S[mb][nt] = X::mma(b, weighted[nt][k], S[mb][nt]);
              }
            }
          }
          if (poisoned) {
            bool hit = false;
            for (int j = 0; j < n; ++j) hit |= (bad[j / 32] >> (j % 32) & 1) && first[p + j] == first_last;
            if (hit) each_state([](float, int, int) { return __builtin_nanf(""); });
            __syncthreads();
            if (threadIdx.x == 0) bad_any = 0;
            __syncthreads();
          }
        }
      }
      fresh = false;
      if (!STATE_ONLY && q.s_out != nullptr && works && seq >= 0 && last[p + n - 1] == begin + n) {
        float* to = q.s_out + (static_cast<int64_t>(seqs[p + n - 1]) * q.heads + head) * q.state_size;
        each_state([&](float s, int i, int j) {
          if (i < q.db && j < q.dc) to[i * q.si + j * q.sj] = s;
          return s;
        });
      }
      p += n;
    }
  }
  if (STATE_ONLY && works) {
    float* to = q.carry + (static_cast<int64_t>(seg) * q.heads + head) * q.db * q.dc;
    each_state([&](float s, int i, int j) {
      if (i < q.db && j < q.dc) to[static_cast<int64_t>(i) * q.dc + j] = s;
      return s;
    });
  }
}

struct Plan {
  int segment, segments;
};

// Segments: as many as give the chip two blocks a compute unit, none shorter than four chunks (a segment costs its share of the first
// pass, and its state is written and read four times).
Plan plan_of(int64_t tokens, int heads, int chunk) {
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  const int64_t want = std::max<int64_t>(1, ceil_div(2 * cus, heads)), chunks = ceil_div(tokens, chunk);
  const int64_t n = std::max<int64_t>(1, std::min(want, chunks / 4));
  Plan p;
  p.segment = static_cast<int>(ceil_div(std::max<int64_t>(chunks, 1), n) * chunk);
  p.segments = static_cast<int>(std::max<int64_t>(1, ceil_div(tokens, p.segment)));
  return p;
}

template <class T, class M, int DBT, int NT>
int launch_mix(const MixArgs& q, hipStream_t st) {
  const uint32_t heads = static_cast<uint32_t>(q.heads);
  if (q.segments > 1) {
    MixArgs own = q;
    own.ga = 1;  // (no outputs, so no a)
    hipLaunchKernelGGL((decay_mix_kernel<T, M, DBT, NT, true>), dim3(static_cast<uint32_t>(q.segments - 1), heads), dim3(kThreads), 0, st, own);
    if (int rc = check_launch("decay_mix_kernel")) return rc;
    const int64_t size = static_cast<int64_t>(q.db) * q.dc;
    hipLaunchKernelGGL(decay_scan_kernel, dim3(static_cast<uint32_t>(ceil_div(size, kScanThreads)), heads), dim3(kScanThreads), 0, st, q);
    if (int rc = check_launch("decay_scan_kernel")) return rc;
  }
  hipLaunchKernelGGL((decay_mix_kernel<T, M, DBT, NT, false>), dim3(static_cast<uint32_t>(q.segments), heads), dim3(kThreads), 0, st, q);
  return check_launch("decay_mix_kernel");
}

template <class T>
int launch_type(const MixArgs& q, hipStream_t st) {
  using M = std::conditional_t<__is_same(T, __bf16), __bf16, float>;  // fp16 goes through fp32 products
  if (q.db <= 64) return q.dc <= 64 ? launch_mix<T, M, 4, 1>(q, st) : launch_mix<T, M, 4, 2>(q, st);
  return q.dc <= 64 ? launch_mix<T, M, 8, 1>(q, st) : launch_mix<T, M, 8, 2>(q, st);
}

struct Layout {
  size_t spans, carry, bytes;
};
Layout layout_of(const ppo_decay_attention_args& a) {
  const int chunk = a.type == PPO_TYPE_BF16 ? Math<__bf16>::CHUNK : Math<float>::CHUNK;
  const Plan p = plan_of(a.tokens, a.kv_heads, chunk);
  Layout l;
  l.spans = 256;
  l.carry = l.spans + (a.cu_seqlens != nullptr ? static_cast<size_t>(ceil_div(a.tokens * sizeof(Span), 256)) * 256 : 0);
  l.bytes = l.carry + static_cast<size_t>(p.segments - 1) * a.kv_heads * a.key_dim * a.value_dim * sizeof(float);
  return l;
}

bool sizes_ok(const ppo_decay_attention_args& a) {
  return a.tokens >= 0 && a.tokens <= INT32_MAX - 65536 && a.sequences >= 1 && a.sequences < INT32_MAX - 1 && a.q_heads >= 1 && a.kv_heads >= 1 &&
         a.q_heads <= 65535 && a.q_heads % a.kv_heads == 0 && a.key_dim >= 1 && a.key_dim <= PPO_DECAY_MAX_DIM && a.value_dim >= 1 &&
         a.value_dim <= PPO_DECAY_MAX_DIM && type_ok(a.type);
}

int check(const char* who, const ppo_decay_attention_args* args, bool backward) {
  PPO_REQUIRE(args != nullptr, "%s: null arguments", who);
  const ppo_decay_attention_args& a = *args;
  PPO_REQUIRE(a.tokens >= 0 && a.tokens <= INT32_MAX - 65536 && a.sequences >= 1 && a.sequences < INT32_MAX - 1, "%s: tokens=%lld sequences=%lld", who,
              (long long)a.tokens, (long long)a.sequences);
  PPO_REQUIRE(a.q_heads >= 1 && a.kv_heads >= 1 && a.q_heads <= 65535 && a.q_heads % a.kv_heads == 0, "%s: q_heads=%d kv_heads=%d", who, a.q_heads, a.kv_heads);
  PPO_REQUIRE(a.key_dim >= 1 && a.key_dim <= PPO_DECAY_MAX_DIM && a.value_dim >= 1 && a.value_dim <= PPO_DECAY_MAX_DIM,
              "%s: key_dim=%d value_dim=%d (1 to %d)", who, a.key_dim, a.value_dim, PPO_DECAY_MAX_DIM);
  PPO_REQUIRE(type_ok(a.type), "%s: type=%d", who, a.type);
  PPO_REQUIRE(a.cu_type == PPO_TOKENS_I64 || a.cu_type == PPO_TOKENS_I32, "%s: cu_type=%d", who, a.cu_type);
  PPO_REQUIRE(a.scale == a.scale && a.scale > -1e30 && a.scale < 1e30, "%s: scale=%g", who, a.scale);
  PPO_REQUIRE(a.cu_seqlens != nullptr || a.sequences == 1, "%s: %lld sequences without cu_seqlens", who, (long long)a.sequences);
  PPO_REQUIRE(a.log_decay != nullptr, "%s: null pointer", who);
  const int64_t n = a.tokens, size = type_size(a.type), hq = a.q_heads, hk = a.kv_heads, dk = a.key_dim, dv = a.value_dim;
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a.log_decay) % 4 == 0 && reinterpret_cast<uintptr_t>(a.initial_state) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(a.final_state) % 4 == 0 && reinterpret_cast<uintptr_t>(a.d_final_state) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(a.d_initial_state) % 4 == 0 &&
                  reinterpret_cast<uintptr_t>(a.cu_seqlens) % (a.cu_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  struct Named {
    const char* name;
    const ppo_head_view* v;
    int64_t heads, dim;
    bool written;
  };
  const Named views[] = {{"q", &a.q, hq, dk, false},        {"k", &a.k, hk, dk, false},      {"v", &a.v, hk, dv, false}, {"out", &a.out, hq, dv, !backward},
                         {"d_q", &a.d_q, hq, dk, true}, {"d_k", &a.d_k, hk, dk, true}, {"d_v", &a.d_v, hk, dv, true}};
  const int count = backward ? 7 : 4;
  for (int i = 0; i < count; ++i)
    if (int rc = check_view(who, views[i].name, *views[i].v, n, views[i].heads, views[i].dim, size, views[i].written)) return rc;
  // every output apart from every input and the other outputs
  const int64_t states = a.sequences * hk * dk * dv * 4;
  struct Region {
    Rows rows;
    int kind;  // 0 read, 1 written
  };
  Region r[16];
  int m = 0;
  for (int i = 0; i < count; ++i)
    if (n > 0) r[m++] = Region{rows_of(*views[i].v, n, views[i].heads, views[i].dim, size), views[i].written};
  r[m++] = Region{vector_of(a.log_decay, hk * 4), 0};
  r[m++] = Region{vector_of(a.cu_seqlens, (a.sequences + 1) * (a.cu_type == PPO_TOKENS_I64 ? 8 : 4)), 0};
  const int in_state = m;
  r[m++] = Region{vector_of(a.initial_state, states), 0};
  r[m++] = Region{vector_of(backward ? a.d_final_state : nullptr, states), 0};
  r[m++] = Region{vector_of(backward ? a.d_initial_state : a.final_state, states), 1};
  for (int i = 0; i < m; ++i)
    for (int k = 0; k < m; ++k) {
      if (r[i].kind != 1 || k == i || (r[k].kind == 1 && k > i)) continue;
      if (i == m - 1 && k == in_state + (backward ? 1 : 0) && r[i].rows.at == r[k].rows.at) continue;  // states in place
      PPO_REQUIRE(!overlap(r[i].rows, r[k].rows), "%s: an output overlaps %s", who, r[k].kind == 1 ? "another" : "an input");
    }
  return PPO_OK;
}

int prepare(const char* who, const ppo_decay_attention_args& a, void* workspace, size_t workspace_bytes, hipStream_t st, MixArgs& q) {
  const Layout l = layout_of(a);
  PPO_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= l.bytes,
              "%s: workspace too small or not 16-byte aligned (%zu < %zu)", who, workspace_bytes, l.bytes);
  const Plan p = plan_of(a.tokens, a.kv_heads, a.type == PPO_TYPE_BF16 ? Math<__bf16>::CHUNK : Math<float>::CHUNK);
  char* base = static_cast<char*>(workspace);
  Span* spans = a.cu_seqlens != nullptr ? reinterpret_cast<Span*>(base + l.spans) : nullptr;
  q = MixArgs{};
  q.log_decay = a.log_decay;
  q.spans = spans;
  q.carry = reinterpret_cast<float*>(base + l.carry);
  q.state_size = static_cast<int64_t>(a.key_dim) * a.value_dim;
  q.tokens = static_cast<int32_t>(a.tokens);
  q.segment = p.segment;
  q.segments = p.segments;
  q.heads = a.kv_heads;
  if (spans != nullptr && a.tokens > 0) {
    hipLaunchKernelGGL(decay_spans_kernel, dim3(static_cast<uint32_t>(ceil_div(a.tokens, kInfoThreads))), dim3(kInfoThreads), 0, st, a.cu_seqlens, a.cu_type,
                       static_cast<int>(a.sequences), q.tokens, spans);
    return check_launch("decay_spans_kernel");
  }
  return PPO_OK;
}

int hand_on(const ppo_decay_attention_args& a, const float* from, float* to, hipStream_t st) {
  if (to == nullptr || from == to) return PPO_OK;
  hipLaunchKernelGGL(decay_empty_kernel, dim3(static_cast<uint32_t>(a.sequences)), dim3(256), 0, st, a.cu_seqlens, a.cu_type, static_cast<int>(a.tokens), from,
                     to, static_cast<int64_t>(a.kv_heads) * a.key_dim * a.value_dim);
  return check_launch("decay_empty_kernel");
}

int mix(const ppo_decay_attention_args& a, const MixArgs& q, hipStream_t st) {
  int rc = PPO_OK;
  with_type(a.type, [&](auto t) { rc = launch_type<decltype(t)>(q, st); });
  return rc;
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_decay_attention_workspace_bytes(const ppo_decay_attention_args* args, int32_t) {
  return args != nullptr && sizes_ok(*args) ? layout_of(*args).bytes : 0;
}

extern "C" int ppo_decay_attention_fwd(const ppo_decay_attention_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream) {
  const char* who = "ppo_decay_attention_fwd";
  if (int rc = check(who, args, false)) return rc;
  const ppo_decay_attention_args& a = *args;
  hipStream_t st = static_cast<hipStream_t>(stream);
  MixArgs q;
  if (int rc = prepare(who, a, workspace, workspace_bytes, st, q)) return rc;
  if (int rc = hand_on(a, a.initial_state, a.final_state, st)) return rc;
  if (a.tokens == 0) return PPO_OK;
  q.a = a.q, q.b = a.k, q.c = a.v, q.out = a.out;
  q.s_in = a.initial_state, q.s_out = a.final_state, q.cut = a.initial_state != nullptr || a.final_state != nullptr;
  q.db = a.key_dim, q.dc = a.value_dim, q.si = a.value_dim, q.sj = 1;
  q.ga = a.q_heads / a.kv_heads, q.gb = 1, q.w = 1;
  q.x = q.y = static_cast<float>(a.scale), q.z = 1.0f;
  return mix(a, q, st);
}

extern "C" int ppo_decay_attention_bwd(const ppo_decay_attention_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream) {
  const char* who = "ppo_decay_attention_bwd";
  if (int rc = check(who, args, true)) return rc;
  const ppo_decay_attention_args& a = *args;
  hipStream_t st = static_cast<hipStream_t>(stream);
  MixArgs q;
  if (int rc = prepare(who, a, workspace, workspace_bytes, st, q)) return rc;
  if (int rc = hand_on(a, a.d_final_state, a.d_initial_state, st)) return rc;
  if (a.tokens == 0) return PPO_OK;
  const int group = a.q_heads / a.kv_heads;
  // d_q: in order, S turned over
  q.a = a.out, q.b = a.v, q.c = a.k, q.out = a.d_q;
  q.s_in = a.initial_state, q.cut = a.initial_state != nullptr;
  q.db = a.value_dim, q.dc = a.key_dim, q.si = 1, q.sj = a.value_dim;
  q.ga = group, q.gb = 1, q.w = 1;
  q.x = q.y = static_cast<float>(a.scale), q.z = 1.0f;
  if (int rc = mix(a, q, st)) return rc;
  // d_k, then d_v, which also hands on the state's gradient: in reverse
  q.reverse = 1, q.w = 0, q.ga = 1, q.gb = group;
  q.x = q.z = static_cast<float>(a.scale), q.y = 1.0f;
  q.s_in = a.d_final_state, q.cut = a.d_final_state != nullptr || a.d_initial_state != nullptr;
  q.a = a.v, q.b = a.out, q.c = a.q, q.out = a.d_k;
  if (int rc = mix(a, q, st)) return rc;
  q.a = a.k, q.b = a.q, q.c = a.out, q.out = a.d_v;
  q.db = a.key_dim, q.dc = a.value_dim, q.si = a.value_dim, q.sj = 1;
  q.s_out = a.d_initial_state;
  return mix(a, q, st);
}
