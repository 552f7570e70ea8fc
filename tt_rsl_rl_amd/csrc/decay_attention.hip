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
// 4 (lane / 16) + 0..3) is that of an operand whose sum runs over those rows, in fours, so S goes into the next product as it lies.  The
// chunk's matrix is made once, its tiles shared out over the waves, and handed round through LDS, where b's rows were: made by each
// wave for itself it took 632 us where this takes 468 (65,536 tokens, 16 heads of 128).  Operands that are sums themselves (S, the matrix,
// weighted c) go into bf16 products as two parts of 8 bits each, which adds 2^-17 to outputs that are rounded to 2^-9 anyway; where a state
// comes out, which is fp32, weighted c has a third part, for 2^-24.  fp16 goes through the fp32 products: a state may leave fp16's
// range, and two bf16 parts of it would need two of q as well.
// With few heads the sequence is cut into segments: a first pass makes each segment's own state, a scan carries them on, and the second pass
// starts every segment from the state before it.
//
// Sequences lie one after another at any offset.  Chunks are cut at multiples of the chunk alone, and the matrix is masked where
// sequences differ; where states come in or go out, chunks are cut at the sequences' ends too.
// A token whose b or c is not finite would reach, as 0 * inf, tokens that do not see it: its row is taken as zeros, and NaN put into
// what does see it.
//
// Bound by what a wave has to issue, at two waves a SIMD: a chunk's matrix products (two and three parts) take a third of the time, the rest goes to splitting
// parts, to LDS and to its barriers.  65,536 tokens of 16 heads of 128 in bf16, states in and out (1.07 GB in and out, 0.2 ms at the copy's rate): 400 us for the
// outputs, 180 for the segments' states, 16 for the scan.
#include <type_traits>

#include "views.hpp"

namespace ppo {
namespace {

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));

constexpr int kInfoThreads = 256;
constexpr int kScanThreads = 256;

// The matrix cores' operand types.  A step sums over K elements, of which a wave's lane group g = lane / 16 holds K / 4 neighbours: one 16-byte
// piece.  An accumulator tile's rows 4 g + 0..3 lie in group g; row_of() says which element a tile's row is, so that QUADS tiles together hold in each
// group the neighbours that the next product's step wants there.
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
  static __device__ __forceinline__ int row_of(int tile, int row) { return 32 * (tile / 2) + 8 * (row / 4) + 4 * (tile % 2) + row % 4; }
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
  static __device__ __forceinline__ int row_of(int tile, int row) { return 16 * tile + row; }
};

// Arrays in LDS: rows of 16-byte pieces, whose places in their row are exchanged by the row's number, so that what a wave reads or writes
// together meets all banks (a read: 16 rows of a tile, four neighbouring pieces; a write: one row, or one piece of rows 8, 4 or 1 apart).
// turn() is made of exclusive ors, so a row that is a lane's part and a constant, without a bit in common, is turned by the one's turn xor the other's:
// from() goes from the lane's place to that of a constant further on with one operation.
template <class M, int ROW_, bool TURNED>
struct Places {
  static constexpr int ROW = ROW_, PIECE = 16 / static_cast<int>(sizeof(M)), PIECES = ROW / PIECE;
  static constexpr __device__ __forceinline__ int turn(int row) {
    return TURNED ? (row >> 1 ^ row >> 4) & 7 : PIECES == 8 ? (row >> 1 ^ (row >> 3 & 2)) & 7 : (row ^ row >> 2) & 15;
  }
  static __device__ __forceinline__ int at(int row, int piece) { return row * ROW + (piece ^ turn(row)) * PIECE; }
  static __device__ __forceinline__ int from(int base, int row, int piece) { return (base ^ (turn(row) ^ piece) * PIECE) + row * ROW; }
};
template <class M, int ROW>  // tokens' rows of ROW elements
using Natural = Places<M, ROW, false>;
template <class M>  // elements' rows of a chunk's tokens: 128 bytes
using Turned = Places<M, Math<M>::CHUNK, true>;

template <class M>
__device__ __forceinline__ typename Math<M>::Frag load_frag(const M* at) {
  return *reinterpret_cast<const typename Math<M>::Frag*>(at);
}

// Values of a step as NP operands whose sum they are, to 8 bits each (bf16; converted in pairs), or as they are (fp32).
template <class M, int NP>
__device__ __forceinline__ void split(float (&x)[4 * Math<M>::QUADS], typename Math<M>::Frag (&out)[NP]) {
  if constexpr (sizeof(M) == 4) {
#pragma unroll
    for (int i = 0; i < 4; ++i) out[0][i] = x[i];
  } else {
    typedef uint32_t Words __attribute__((ext_vector_type(4)));
    typedef __bf16 Pair __attribute__((ext_vector_type(2)));
#pragma unroll
    for (int p = 0; p < NP; ++p) {
      Words w;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const Pair pair{static_cast<__bf16>(x[2 * i]), static_cast<__bf16>(x[2 * i + 1])};
        w[i] = __builtin_bit_cast(uint32_t, pair);
        if (p + 1 < NP) {
          x[2 * i] -= __builtin_bit_cast(float, w[i] << 16);
          x[2 * i + 1] -= __builtin_bit_cast(float, w[i] & 0xffff0000u);
        }
      }
      out[p] = __builtin_bit_cast(typename Math<M>::Frag, w);
    }
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
  float* carry;         // [segments - 1][heads][elements]: the state that leaves a segment, then what enters the next; element (i, j) at i * ci + j * cj
  int64_t si, sj, state_size;
  int32_t ci, cj;
  int32_t carried;      // carry holds what enters the segments already
  int32_t exact;        // states come out, in fp32: three parts of what makes them
  int32_t tokens, segment, segments;
  int32_t heads, ga, gb;  // heads of b, c and S times gb; of a per head and block
  int32_t spread;         // blocks that share a's heads of a head
  int32_t db, dc;
  int32_t reverse, w, cut;  // cut: chunks end with their sequence
  int32_t near;             // the outputs' rows too, and aligned to four bytes
  int32_t whole;            // rows are whole 16-byte pieces, not far apart
  float x, y, z;
};

__device__ __forceinline__ Span span_of(const MixArgs& q, int token) {
  return q.spans == nullptr ? Span{0, q.tokens, 0} : q.spans[token];
}

struct SequenceArgs {
  const void* cu;
  int32_t cu_type, tokens;
  int64_t sequences;
  Span* spans;  // of each token, by the first token_blocks blocks
  int64_t token_blocks;
  const float* from;  // the states of sequences without tokens, or of all, by the others
  float* to;
  int64_t size;
  int32_t all;
};

// What chunks do not do: one thread a token, the sequence that it lies in; one block a sequence, its state handed on.
__global__ __launch_bounds__(kInfoThreads) void decay_sequences_kernel(const SequenceArgs q) {
  auto at = [&](int64_t i) {
    return q.cu_type == PPO_TOKENS_I64 ? static_cast<const int64_t*>(q.cu)[i] : static_cast<int64_t>(static_cast<const int32_t*>(q.cu)[i]);
  };
  const int64_t tokens = q.tokens;
  if (blockIdx.x >= q.token_blocks) {
    for (int64_t b = blockIdx.x - q.token_blocks; b < q.sequences; b += gridDim.x - q.token_blocks) {
      const bool empty = q.cu == nullptr ? tokens == 0 : min(at(b + 1), tokens) <= max(at(b), static_cast<int64_t>(0));
      if (!empty && q.all == 0) continue;
      for (int64_t i = threadIdx.x; i < q.size; i += kInfoThreads) q.to[b * q.size + i] = q.from == nullptr ? 0.0f : q.from[b * q.size + i];
    }
    return;
  }
  const int64_t t = static_cast<int64_t>(blockIdx.x) * kInfoThreads + threadIdx.x;
  if (t >= tokens) return;
  int64_t lo = 0, hi = q.sequences + 1;  // the first entry above t
  while (lo < hi) {
    const int64_t mid = (lo + hi) / 2;
    if (at(mid) > t) hi = mid;
    else lo = mid + 1;
  }
  Span s{static_cast<int32_t>(t), static_cast<int32_t>(t) + 1, -1};
  if (lo >= 1 && lo <= q.sequences) {
    const int64_t from = max(at(lo - 1), static_cast<int64_t>(0)), to = min(at(lo), tokens);
    if (from <= t && to > t) s = Span{static_cast<int32_t>(from), static_cast<int32_t>(to), static_cast<int32_t>(lo - 1)};
  }
  q.spans[t] = s;
}

// carry[s] holds what segment s makes of nothing; afterwards what enters segment s + 1.
__global__ __launch_bounds__(kScanThreads) void decay_scan_kernel(const MixArgs q) {
  const int64_t size = q.state_size, i = static_cast<int64_t>(blockIdx.x) * kScanThreads + threadIdx.x;
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

// Whether any of the values is not finite: 0 x is 0 but for those.
template <class T>
__device__ __forceinline__ float sum_of_nothing(const RawPiece& r, float sum) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if constexpr (sizeof(T) == 4) {
      sum = fmaf(__builtin_bit_cast(float, r.w[i]), 0.0f, sum);
    } else if constexpr (__is_same(T, __bf16)) {
      typedef __bf16 Two __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(Two, r.w[i]), Two{}, sum, false);
    } else {
      typedef _Float16 Two __attribute__((ext_vector_type(2)));
      sum = __builtin_amdgcn_fdot2(__builtin_bit_cast(Two, r.w[i]), Two{}, sum, false);
    }
  }
  return sum;
}
template <class T>
__device__ __forceinline__ bool not_finite(const RawPiece& r) { return !(sum_of_nothing<T>(r, 0.0f) == 0.0f); }
template <class T>
__device__ __forceinline__ bool not_finite(const RawPiece (&r)[4]) {
  float sum = 0.0f;
#pragma unroll
  for (int k = 0; k < 4; ++k) sum = sum_of_nothing<T>(r[k], sum);
  return !(sum == 0.0f);
}

// Four tokens' pieces of 16 bytes, columns d .., into rows of tokens and into rows of elements.
template <class T, class M, int ROW>
__device__ __forceinline__ void put_rows(const RawPiece (&r)[4], M* rows, int j4, int d, bool there) {
  typedef Natural<M, ROW> N;
  constexpr int V = kVec<T>;
  const int base = N::at(j4, d / N::PIECE);
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    if constexpr (sizeof(T) == sizeof(M)) {
      RawPiece x;
#pragma unroll
      for (int i = 0; i < 4; ++i) x.w[i] = there ? r[k].w[i] : 0;
      *reinterpret_cast<RawPiece*>(rows + N::from(base, k, 0)) = x;
    } else {
#pragma unroll
      for (int e = 0; e < V; e += 4) {
        f32x4 x;
#pragma unroll
        for (int f = 0; f < 4; ++f) x[f] = there ? element<T>(r[k], e + f) : 0.0f;
        *reinterpret_cast<f32x4*>(rows + N::from(base, k, e / 4)) = x;
      }
    }
  }
}

template <class T, class M>
__device__ __forceinline__ void put_turned(const RawPiece (&r)[4], M* turned, int j4, int d) {
  typedef Turned<M> N;
  constexpr int V = kVec<T>;
  const int base = N::at(d, j4 / N::PIECE) + j4 % N::PIECE;
#pragma unroll
  for (int e = 0; e < V; ++e) {
    typename Math<M>::Quad x;
    if constexpr (sizeof(M) == 2) {
      typedef uint32_t Two __attribute__((ext_vector_type(2)));
      const uint32_t pick = e % 2 != 0 ? 0x07060302u : 0x05040100u;  // the high, the low halves
      x = __builtin_bit_cast(typename Math<M>::Quad, Two{__builtin_amdgcn_perm(r[1].w[e / 2], r[0].w[e / 2], pick),
                                                         __builtin_amdgcn_perm(r[3].w[e / 2], r[2].w[e / 2], pick)});
    } else {
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] = static_cast<M>(element<T>(r[k], e));
    }
    *reinterpret_cast<typename Math<M>::Quad*>(turned + N::from(base, e, 0)) = x;
  }
}

// T: the views' type, M: the products', DBT: tiles of 16 of b's elements, NT: tiles of 16 of c's elements to each of four waves, STATE_ONLY:
// the first pass over segments, which makes their own states.
//
// A block goes through items: a piece of up to CHUNK tokens (times the heads that share it).  An item's rows are loaded into registers while
// the item before is computed.
constexpr int kWaves = 4;
constexpr int kThreads = kWaves * kWave;

// A raw buffer of 2 GiB at a wave-uniform address.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0, 0x7fffffff, 0x00020000);
}

// Everything on its way from and to memory has arrived.  At the end of a branch that is rarely taken: where paths meet, the compiler otherwise waits, at the first use of
// what one of them loaded, for everything that was issued since on any, the next item's rows among it (65,536 tokens of 16 heads of 128: 427 us so, 391
// with these waits and stores that are always issued).
__device__ __forceinline__ void wait_memory() { __builtin_amdgcn_s_waitcnt(0x0f70); }

template <class T, class M, int DBT, int NT, bool STATE_ONLY>
__global__ __launch_bounds__(kThreads, 2) void decay_mix_kernel(const MixArgs q) {
  typedef Math<M> X;
  typedef typename X::Frag Frag;
  static_assert(2 * kWaves * 16 >= PPO_DECAY_MAX_DIM);
  constexpr int C = X::CHUNK, K = X::K, Q = X::QUADS, DB = DBT * 16, DC = kWaves * NT * 16, IT = C / 16, V = kVec<T>;
  constexpr int PARTS = X::PARTS2;
  typedef Natural<M, DB> Rows_;
  typedef Turned<M> Cols_;
  constexpr int B_ROWS = C * DB > PARTS * C * C ? C * DB : PARTS * C * C;
  __shared__ __align__(16) M a_rows[STATE_ONLY ? 8 : C * DB];
  __shared__ __align__(16) M b_rows[STATE_ONLY ? 8 : B_ROWS];  // then the chunk's matrix, [part][i][j]
  __shared__ __align__(16) M b_turned[DB * C];
  __shared__ __align__(16) M c_turned[DC * C];
  __shared__ __align__(16) float weights[C], sights[C];  // of each token in the next state; of the state before in each output
  __shared__ float fades[C + 1];
  __shared__ int first[2][C], last[2][C], seqs[2][C];  // of the chunk's tokens and the next one's
  __shared__ uint32_t bad_any, bad[(C + 31) / 32];

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int head = blockIdx.y, seg = blockIdx.x;
  const int columns = NT == 1 && q.dc > DC ? 2 : 1, share = blockIdx.z / columns, col0 = blockIdx.z % columns * DC;  // a block has DC of c's columns
  const int a_head = (head * q.spread + share) * q.ga;
  const int own0 = wave * NT * 16, dc0 = col0 + own0;
  const bool works = dc0 < q.dc;
  const int seg_begin = seg * q.segment, seg_end = min(seg_begin + q.segment, q.tokens);

  f32x4 S[DBT][NT];  // rows row_of(mb, 4 g + 0..3), column column_of(nt)
  // Where a lane owns outputs' elements: with two tiles 8 neighbours, so that they leave in 16 bytes.
  auto column_of = [](int nt, int col) { return NT == 2 ? 8 * (col / 4) + 4 * nt + col % 4 : col; };
  auto each_state = [&](auto&& f) {
    int group = 4 * (lane / 16), col = lane % 16;
    forget(group), forget(col);  // (or else every element's address is kept from one chunk to the next, in 128 registers)
#pragma unroll
    for (int mb = 0; mb < DBT; ++mb)
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int r = 0; r < 4; ++r) S[mb][nt][r] = f(S[mb][nt][r], X::row_of(mb, group + r), dc0 + column_of(nt, col));
  };
  auto token_at_place = [&](int u) { return q.reverse ? q.tokens - 1 - u : u; };
  auto put_span = [&](int buffer, int u, const Span& s) {  // positions in the order that is walked
    const int i = threadIdx.x;
    first[buffer][i] = q.reverse ? q.tokens - s.end : s.start;
    last[buffer][i] = q.reverse ? q.tokens - s.start : s.end;
    seqs[buffer][i] = s.seq;
  };

  // An item's rows: units of four tokens by 16 bytes, first b's, then c's, then a's; a wave's 64 are of one view.  What is loaded past the
  // last token is that token again: it has no weight anywhere.
  constexpr int UB = DB / V * (C / 4), UC = DC / V * (C / 4), UA = STATE_ONLY ? 0 : UB, ROUNDS = (UB + UC + UA + kThreads - 1) / kThreads;
  static_assert(UB % kWave == 0 && UC % kWave == 0);
  RawPiece r[ROUNDS][4];
  auto kind_of = [&](int round) {  // 0: b, 1: c, 2: a, 3: none
    const int i = (round * kWaves + wave) * kWave;
    return i < UB ? 0 : i < UB + UC ? 1 : i < UB + UC + UA ? 2 : 3;
  };
  auto place_of = [&](int thread, int round, int kind, int& j4, int& d) {
    const int i = thread + round * kThreads - (kind == 0 ? 0 : kind == 1 ? UB : UB + UC);
    const int pieces = (kind == 1 ? DC : DB) / V;
    j4 = i / pieces % (C / 4) * 4;
    d = i % pieces * V;
  };
  auto load_rows = [&](int begin, int n, int ab) {
    const int ha = q.ga > 1 ? a_head + ab : a_head, hb = q.gb > 1 ? head * q.gb + ab : head;
    const int64_t lowest = q.reverse ? q.tokens - begin - n : begin;
    int thread = threadIdx.x;
    forget(thread);  // (addresses again)
#pragma unroll
    for (int round = 0; round < ROUNDS; ++round) {
      const int kind = kind_of(round);
      int j4, d;
      place_of(thread, round, kind, j4, d);
      const ppo_head_view& v = kind == 0 ? q.b : kind == 1 || STATE_ONLY ? q.c : q.a;
      const char* from = reinterpret_cast<const char*>(static_cast<const T*>(v.data) + (kind >= 2 ? ha : hb) * v.head_stride + lowest * v.token_stride);
      const uint32_t step = static_cast<uint32_t>(v.token_stride) * sizeof(T);
      const uint32_t column = min(d + (kind == 1 || (STATE_ONLY && kind == 3) ? col0 : 0), (kind == 1 || (STATE_ONLY && kind == 3) ? q.dc : q.db) - V) * static_cast<int>(sizeof(T));
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        const int j = min(j4 + k, n - 1);
        r[round][k] = load_raw(reinterpret_cast<const T*>(from + (__umul24(q.reverse ? n - 1 - j : j, step) + column)));
      }
    }
  };

  if (threadIdx.x <= C) fades[threadIdx.x] = threadIdx.x == 0 ? 1.0f : static_cast<float>(exp(static_cast<double>(q.log_decay[head]) * threadIdx.x));
  if (threadIdx.x == 0) bad_any = 0;
  if (threadIdx.x < (C + 31) / 32) bad[threadIdx.x] = 0;
  if (seg_begin + static_cast<int>(threadIdx.x) < min(seg_begin + C, seg_end))
    put_span(0, seg_begin + threadIdx.x, span_of(q, token_at_place(seg_begin + threadIdx.x)));
  lds_barrier();
  bool fresh = true;  // S is zeros
  each_state([](float, int, int) { return 0.0f; });
  if (!STATE_ONLY && first[0][0] < seg_begin) {  // goes on from the segment before
    const float* from = q.carry + (static_cast<int64_t>(seg - 1) * q.heads + head) * q.state_size;
    each_state([&](float, int i, int j) { return works && i < q.db && j < q.dc ? from[i * q.ci + j * q.cj] : 0.0f; });
    wait_memory();
    fresh = false;
  }

  int c0 = seg_begin, p = 0, ab = 0, buffer = 0;  // the item: chunk, place in it, head
  auto length = [&](int b, int at, int chunk) {
    const int cn = min(C, seg_end - chunk);
    return __builtin_amdgcn_readfirstlane(q.cut ? min(cn - at, last[b][at] - (chunk + at)) : cn - at);
  };
  int n = length(0, 0, c0);
  if (q.whole) load_rows(c0, n, 0);
  f32x4 acc[IT][NT];
  const int abs = q.ga * q.gb;
  while (true) {
    const int begin = c0 + p, seq = __builtin_amdgcn_readfirstlane(seqs[buffer][p]), first0 = __builtin_amdgcn_readfirstlane(first[buffer][p]);
    const int first_last = __builtin_amdgcn_readfirstlane(first[buffer][p + n - 1]);  // where the sequence of the last token begins
    const int* const from_first = first[buffer] + p;
    const uint64_t valid = __ballot(lane < n && seqs[buffer][p + min(lane, n - 1)] >= 0);  // tokens of sequences
    const bool new_b = q.gb > 1 || ab == 0, new_a = !STATE_ONLY && (q.ga > 1 || ab == 0);
    const bool ahead = ab == 0 && p == 0 && c0 + C + static_cast<int>(threadIdx.x) < min(c0 + 2 * C, seg_end);
    Span next_span{};
    if (ahead) next_span = span_of(q, token_at_place(c0 + C + threadIdx.x));
    if (ab == 0 && first0 == begin) {  // a sequence begins
      fresh = q.s_in == nullptr || seq < 0;
      const float* from = q.s_in + (static_cast<int64_t>(seq) * q.heads + head) * q.state_size;
      if (fresh) each_state([](float, int, int) { return 0.0f; });
      else each_state([&](float, int i, int j) { return works && i < q.db && j < q.dc ? from[i * q.si + j * q.sj] : 0.0f; });
      wait_memory();
    }
    int thread = threadIdx.x;
    forget(thread);
    const int col = thread % 16, g = thread % kWave / 16;
    const int a_at = Rows_::at(col, g), b_at = Rows_::at(X::row_of(0, col), g), m_at = Cols_::at(col, g), bt_at = Cols_::at(X::row_of(0, col), g);
    const int ct_at = Cols_::at(own0 + column_of(0, col), g);  // operands' places, to go on from
    // ---- rows into LDS ----
    lds_barrier();  // the last products have read what is there
    if (q.whole) {
#pragma unroll
      for (int round = 0; round < ROUNDS; ++round) {
        const int kind = kind_of(round);
        int j4, d;
        place_of(thread, round, kind, j4, d);
        if (kind < 2 && not_finite<T>(r[round])) {
#pragma unroll
          for (int k = 0; k < 4; ++k)
            if (not_finite<T>(r[round][k])) atomicOr(&bad[(j4 + k) / 32], 1u << ((j4 + k) % 32));
          bad_any = 1;
        }
        if (!STATE_ONLY && kind == 0) put_rows<T, M, DB>(r[round], b_rows, j4, d, true);  // (b's rows have made room for the last matrix)
        if (kind == 0 && new_b) put_turned<T, M>(r[round], b_turned, j4, d);
        if (kind == 1 && new_b) put_turned<T, M>(r[round], c_turned, j4, d);
        // (past b's elements a is zeros, and what b and S hold there is not seen)
        if (!STATE_ONLY && kind == 2 && new_a) put_rows<T, M, DB>(r[round], a_rows, j4, d, d < q.db);
      }
    } else {  // heads of odd widths: element by element
      auto elements = [&](const ppo_head_view& v, int h, int dim, int from, int padded, M* rows, M* turned) {
        constexpr int AHEAD = 8;  // loads in flight, of what is there (one at a time 700 tokens of 8 heads of 10 and 13 took 204 us going back, so 150)
        static_assert(C * 64 % (kThreads * AHEAD) == 0);
#pragma unroll 1
        for (int i0 = thread; i0 < C * padded; i0 += kThreads * AHEAD) {
          T x[AHEAD];
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * kThreads, j = min(i / padded, n - 1), d = min(from + i % padded, dim - 1);
            x[u] = static_cast<const T*>(v.data)[h * v.head_stride + token_at_place(begin + j) * v.token_stride + d];
          }
#pragma unroll
          for (int u = 0; u < AHEAD; ++u) {
            const int i = i0 + u * kThreads, j = i / padded, d = i % padded;
            const T y = from + d < dim && (valid >> j & 1) != 0 ? x[u] : static_cast<T>(0.0f);
            if (turned != nullptr && !(fabsf(static_cast<float>(y)) < INFINITY)) {
              atomicOr(&bad[j / 32], 1u << (j % 32));
              bad_any = 1;
            }
            if (rows != nullptr) rows[Rows_::at(j, d / Rows_::PIECE) + d % Rows_::PIECE] = static_cast<M>(y);
            if (turned != nullptr) turned[Cols_::at(d, j / Cols_::PIECE) + j % Cols_::PIECE] = static_cast<M>(y);
          }
        }
      };
      const int ha = q.ga > 1 ? a_head + ab : a_head, hb = q.gb > 1 ? head * q.gb + ab : head;
      if (new_a) elements(q.a, ha, q.db, 0, DB, a_rows, nullptr);
      elements(q.b, hb, q.db, 0, DB, STATE_ONLY ? nullptr : b_rows, b_turned);
      if (new_b) elements(q.c, hb, q.dc, col0, DC, nullptr, c_turned);
    }
    if (thread < C) {
      const int i = min(thread, n - 1);
      weights[thread] = thread < n && from_first[i] == first_last ? q.z * fades[n - q.w - i] : 0.0f;
      sights[thread] = thread < n && from_first[i] == first0 ? q.y * fades[i + q.w] : __builtin_nanf("");  // (NaN: not at all)
    }
    if (ahead) put_span(buffer ^ 1, c0 + C + threadIdx.x, next_span);
    wait_memory();  // (the spans, as the compiler sees it, on the path that did not load them)
    lds_barrier();
    const bool poisoned = __builtin_amdgcn_readfirstlane(bad_any) != 0;
    if (poisoned) {  // zeros where a token is not finite, and in the places behind the last one, which hold it too
      for (int j = 0; j < C; ++j)
        if (bad[j / 32] >> (j % 32) & 1) {
          for (int d = thread; d < DB; d += kThreads) {
            if (!STATE_ONLY) b_rows[Rows_::at(j, d / Rows_::PIECE) + d % Rows_::PIECE] = static_cast<M>(0.0f);
            b_turned[Cols_::at(d, j / Cols_::PIECE) + j % Cols_::PIECE] = static_cast<M>(0.0f);
          }
          for (int d = thread; d < DC; d += kThreads) c_turned[Cols_::at(d, j / Cols_::PIECE) + j % Cols_::PIECE] = static_cast<M>(0.0f);
        }
      lds_barrier();
    }
    // ---- the next item, and its rows on their way ----
    int next_ab = ab + 1, next_p = p, next_c0 = c0, next_buffer = buffer, next_n = n;
    if (next_ab == abs) {
      next_ab = 0, next_p = p + n;
      if (next_p >= min(C, seg_end - c0)) next_p = 0, next_c0 = c0 + C, next_buffer = buffer ^ 1;
      if (next_c0 < seg_end) next_n = length(next_buffer, next_p, next_c0);
    }
    const bool done = next_c0 >= seg_end;
    if (q.whole) load_rows(done ? begin : next_c0 + next_p, next_n, done ? ab : next_ab);  // (once more at the end: loads without a branch stay in their registers)

    if constexpr (!STATE_ONLY) {
      // ---- the chunk's matrix, its steps of tiles with i >= j shared among the waves ----
      {
        constexpr int EACH = kWaves / IT, STEPS = (C / K + EACH - 1) / EACH;
        const int it = wave / EACH, step0 = wave % EACH, i = 16 * it + col;
        Frag matrix[STEPS][PARTS];
        Frag a[DB / K];
#pragma unroll
        for (int ks = 0; ks < DB / K; ++ks) a[ks] = load_frag<M>(a_rows + Rows_::from(a_at, 16 * it, 4 * ks));
        const int lowest = i < n ? from_first[min(i, n - 1)] - begin : C;  // the first of the piece's tokens that i sees
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
          const int kj = step0 + step * EACH;
          if (kj * Q > it) continue;
          float v[4 * Q];
#pragma unroll
          for (int h = 0; h < Q; ++h) {
            const int jt = kj * Q + h;
            f32x4 m{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int ks = 0; ks < DB / K; ++ks) m = X::mma(load_frag<M>(b_rows + Rows_::from(b_at, X::row_of(jt, 0), 4 * ks)), a[ks], m);
            const int j0 = X::row_of(jt, 4 * g);
            float f[4];
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) f[r4] = fades[max(i - j0 - r4, 0)];
            asm volatile("" : "+v"(f[0]), "+v"(f[1]), "+v"(f[2]), "+v"(f[3]));  // (or else each is read in a branch, with a wait)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) v[4 * h + r4] = (j0 + r4 <= i) & (j0 + r4 >= lowest) ? m[r4] * (q.x * f[r4]) : 0.0f;
          }
          split<M, PARTS>(v, matrix[step]);
        }
        lds_barrier();  // b's rows have been read
#pragma unroll
        for (int step = 0; step < STEPS; ++step) {
          const int kj = step0 + step * EACH;
          if (kj * Q > it) continue;
#pragma unroll
          for (int k = 0; k < PARTS; ++k) *reinterpret_cast<Frag*>(b_rows + k * C * C + Cols_::from(m_at, 16 * it, 4 * kj)) = matrix[step][k];
        }
      }
      // ---- what lies before the piece ----
      if (ab == 0 || q.ga > 1) {
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) acc[i][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        if (works && !fresh) {
#pragma unroll
          for (int ks = 0; ks < DB / K; ++ks) {
            Frag s[NT][PARTS];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
              float v[4 * Q];
#pragma unroll
              for (int i = 0; i < 4 * Q; ++i) v[i] = S[ks * Q + i / 4][nt][i % 4];
              split<M, PARTS>(v, s[nt]);
            }
#pragma unroll
            for (int i = 0; i < IT; ++i) {
              const Frag a = load_frag<M>(a_rows + Rows_::from(a_at, 16 * i, 4 * ks));
#pragma unroll
              for (int k = 0; k < PARTS; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) acc[i][nt] = X::mma(s[nt][k], a, acc[i][nt]);
            }
          }
#pragma unroll
          for (int i = 0; i < IT; ++i) {
            const float f = sights[16 * i + col];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r4 = 0; r4 < 4; ++r4) acc[i][nt][r4] = f == f ? acc[i][nt][r4] * f : 0.0f;  // (0 times what is not finite is not finite)
          }
        }
      }
      lds_barrier();  // the matrix is there
    }
    if (works) {
      Frag c[NT][C / K];  // c's columns that the wave owns
#pragma unroll
      for (int nt = 0; nt < NT; ++nt)
#pragma unroll
        for (int kj = 0; kj < C / K; ++kj) c[nt][kj] = load_frag<M>(c_turned + Cols_::from(ct_at, column_of(nt, 0), 4 * kj));
      if constexpr (!STATE_ONLY) {
        // ---- the piece's tokens among each other ----
#pragma unroll
        for (int i = 0; i < IT; ++i)
#pragma unroll
          for (int kj = 0; kj < C / K; ++kj) {
            if (kj * Q > i) continue;
#pragma unroll
            for (int k = 0; k < PARTS; ++k) {
              const Frag m = load_frag<M>(b_rows + k * C * C + Cols_::from(m_at, 16 * i, 4 * kj));
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[i][nt] = X::mma(c[nt][kj], m, acc[i][nt]);
            }
          }
        if (poisoned)
#pragma unroll
          for (int i = 0; i < IT; ++i) {
            const int at = 16 * i + col, mine = from_first[min(at, n - 1)];
            bool hit = false;
            for (int j = 0; j <= min(at, n - 1); ++j) hit |= (bad[j / 32] >> (j % 32) & 1) && from_first[j] == mine;
            if (hit)
#pragma unroll
              for (int nt = 0; nt < NT; ++nt) acc[i][nt] = f32x4{__builtin_nanf(""), __builtin_nanf(""), __builtin_nanf(""), __builtin_nanf("")};
          }
        // ---- the outputs ----
        if (q.ga > 1 || ab == q.gb - 1) {
          const int ha = q.ga > 1 ? a_head + ab : a_head, d = dc0 + 4 * NT * g;
          const int64_t lowest = q.reverse ? q.tokens - begin - n : begin;
          T* const to = static_cast<T*>(q.out.data) + ha * q.out.head_stride + lowest * q.out.token_stride;
          if (q.near) {
            // stores that are always issued: a row that is none goes past the buffer's end, where nothing is written
            const auto buffer = buffer_at(to);
            const uint32_t step = static_cast<uint32_t>(q.out.token_stride) * sizeof(T);
#pragma unroll
            for (int i = 0; i < IT; ++i) {
              const int at = 16 * i + col;
              const uint32_t off = (valid >> at & 1) != 0 && d < q.dc ? __umul24(q.reverse ? n - 1 - at : at, step) + d * static_cast<uint32_t>(sizeof(T)) : 0x80000000u;
              typedef uint32_t Words __attribute__((ext_vector_type(4)));
              typedef T Piece16 __attribute__((ext_vector_type(16 / sizeof(T))));
              constexpr int PER = 16 / static_cast<int>(sizeof(T));
              if constexpr (4 * NT * sizeof(T) >= 16) {
#pragma unroll
                for (int e = 0; e < 4 * NT; e += PER) {
                  Piece16 o;
#pragma unroll
                  for (int f = 0; f < PER; ++f) o[f] = static_cast<T>(acc[i][(e + f) / 4][(e + f) % 4]);
                  // (of fp32's two pieces the first may be the head's last)
                  const uint32_t piece = e == 0 || d + e < q.dc ? off + e * static_cast<uint32_t>(sizeof(T)) : 0x80000000u;
                  __builtin_amdgcn_raw_buffer_store_b128(__builtin_bit_cast(Words, o), buffer, piece, 0, 0);
                }
              } else {
                typedef uint32_t Pair __attribute__((ext_vector_type(2)));
                typedef T Four __attribute__((ext_vector_type(4)));
                Four o;
#pragma unroll
                for (int f = 0; f < 4; ++f) o[f] = static_cast<T>(acc[i][0][f]);
                __builtin_amdgcn_raw_buffer_store_b64(__builtin_bit_cast(Pair, o), buffer, off, 0, 0);
              }
            }
          } else {
#pragma unroll
            for (int i = 0; i < IT; ++i) {
              const int at = 16 * i + col;
              if (valid >> at & 1) {
                T* row = to + (static_cast<uint64_t>(static_cast<uint32_t>(q.reverse ? n - 1 - at : at)) * static_cast<uint32_t>(q.out.token_stride) + d);
#pragma unroll
                for (int e = 0; e < 4 * NT; ++e)
                  if (d + e < q.dc) row[e] = static_cast<T>(acc[i][e / 4][e % 4]);
              }
            }
            wait_memory();
          }
        }
      }
      // ---- the state ----
      if (ab >= q.ga - 1) {
        if (ab == q.ga - 1) {
          const float f = fades[n];
#pragma unroll
          for (int mb = 0; mb < DBT; ++mb)
#pragma unroll
            for (int nt = 0; nt < NT; ++nt)
#pragma unroll
              for (int r4 = 0; r4 < 4; ++r4) S[mb][nt][r4] *= f;
          if (first_last != first0) each_state([](float, int, int) { return 0.0f; });  // another sequence's, which may have left fp32's range
        }
#pragma unroll
        for (int kj = 0; kj < C / K; ++kj) {
          f32x4 w[Q];
#pragma unroll
          for (int h = 0; h < Q; ++h) w[h] = *reinterpret_cast<const f32x4*>(weights + K * kj + K / 4 * g + 4 * h);
          Frag weighted[NT][X::PARTS3];
#pragma unroll
          for (int nt = 0; nt < NT; ++nt) {
            float v[4 * Q];
#pragma unroll
            for (int i = 0; i < 4 * Q; ++i) v[i] = w[i / 4][i % 4] * static_cast<float>(c[nt][kj][i]);
            split<M, X::PARTS3>(v, weighted[nt]);
          }
          auto add = [&](auto parts_from, auto parts_to) {
#pragma unroll
            for (int mb = 0; mb < DBT; ++mb) {
              const Frag b = load_frag<M>(b_turned + Cols_::from(bt_at, X::row_of(mb, 0), 4 * kj));
#pragma unroll
              for (int k = parts_from; k < parts_to; ++k)
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) S[mb][nt] = X::mma(b, weighted[nt][k], S[mb][nt]);
            }
          };
          constexpr int two = X::PARTS3 < 2 ? X::PARTS3 : 2;
          add(std::integral_constant<int, 0>{}, std::integral_constant<int, two>{});
          if (two < X::PARTS3 && q.exact) add(std::integral_constant<int, two>{}, std::integral_constant<int, X::PARTS3>{});
        }
      }
    }
    if (poisoned && ab >= q.ga - 1) {
      bool hit = false;
      for (int j = 0; j < n; ++j) hit |= (bad[j / 32] >> (j % 32) & 1) && from_first[j] == first_last;
      if (hit) each_state([](float, int, int) { return __builtin_nanf(""); });
      lds_barrier();
      if (threadIdx.x == 0) bad_any = 0;
      if (threadIdx.x < (C + 31) / 32) bad[threadIdx.x] = 0;
    }
    if (ab == abs - 1) {
      fresh = false;
      if (!STATE_ONLY && q.s_out != nullptr && share == 0 && works && seq >= 0 && last[buffer][p + n - 1] == begin + n) {
        float* to = q.s_out + (static_cast<int64_t>(seqs[buffer][p + n - 1]) * q.heads + head) * q.state_size;
        each_state([&](float s, int i, int j) {
          if (i < q.db && j < q.dc) to[i * q.si + j * q.sj] = s;
          return s;
        });
      }
    }
    if (done) break;
    c0 = next_c0, p = next_p, ab = next_ab, buffer = next_buffer, n = next_n;
  }
  if (STATE_ONLY && works) {
    float* to = q.carry + (static_cast<int64_t>(seg) * q.heads + head) * q.state_size;
    each_state([&](float s, int i, int j) {
      if (i < q.db && j < q.dc) to[i * q.ci + j * q.cj] = s;
      return s;
    });
  }
}

struct Plan {
  int segment, segments;
};

// Segments: as many as give the chip two blocks a compute unit (a segment's state is written and read four times), down to a chunk each: a block alone
// on its compute unit takes 5 to 7 us a chunk, waiting (577 tokens of 3 heads, fp32, the whole call: segments of four chunks 120 us, of one 47).
// Where states make a piece of each sequence, segments go down to the sequences' mean length (14 sequences of a token, 12 heads: 79 us as one segment, 47 so).
Plan plan_of(const ppo_decay_attention_args& a) {
  const int chunk = a.type == PPO_TYPE_BF16 ? Math<__bf16>::CHUNK : Math<float>::CHUNK;
  const bool states = a.initial_state != nullptr || a.final_state != nullptr || a.d_final_state != nullptr || a.d_initial_state != nullptr;
  const int64_t least = states ? std::min<int64_t>(std::max<int64_t>(a.tokens / a.sequences, 1), chunk) : chunk;
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  const int64_t want = std::max<int64_t>(1, ceil_div(2 * cus, a.kv_heads)), pieces = ceil_div(a.tokens, least);
  const int64_t n = std::max<int64_t>(1, std::min(want, pieces));
  Plan p;
  p.segment = static_cast<int>(ceil_div(std::max<int64_t>(pieces, 1), n) * least);
  p.segments = static_cast<int>(std::max<int64_t>(1, ceil_div(a.tokens, p.segment)));
  return p;
}

template <class T, class M, int DBT, int NT>
int launch_mix(const MixArgs& q, hipStream_t st) {
  const uint32_t heads = static_cast<uint32_t>(q.heads), columns = static_cast<uint32_t>(ceil_div(q.dc, kWaves * NT * 16));
  if (q.segments > 1 && q.carried == 0) {
    MixArgs own = q;
    own.ga = own.spread = 1;  // (no outputs, so no a)
    hipLaunchKernelGGL((decay_mix_kernel<T, M, DBT, NT, true>), dim3(static_cast<uint32_t>(q.segments - 1), heads, columns), dim3(kThreads), 0, st, own);
    if (int rc = check_launch("decay_mix_kernel")) return rc;
    const int64_t size = static_cast<int64_t>(q.db) * q.dc;
    hipLaunchKernelGGL(decay_scan_kernel, dim3(static_cast<uint32_t>(ceil_div(size, kScanThreads)), heads), dim3(kScanThreads), 0, st, q);
    if (int rc = check_launch("decay_scan_kernel")) return rc;
  }
  // a's heads one to a block, or a few, where that many blocks still find a compute unit each (the same tokens, 6 query heads: 22 us together, 15 so)
  MixArgs whole = q;
  whole.spread = q.ga;
  while (whole.spread > 1 && (q.ga % whole.spread != 0 || static_cast<int64_t>(q.segments) * heads * columns * whole.spread > device_info().cus)) --whole.spread;
  whole.ga = q.ga / whole.spread;
  hipLaunchKernelGGL((decay_mix_kernel<T, M, DBT, NT, false>), dim3(static_cast<uint32_t>(q.segments), heads, columns * whole.spread), dim3(kThreads), 0, st, whole);
  return check_launch("decay_mix_kernel");
}

template <class T>
int launch_type(const MixArgs& q, hipStream_t st) {
  using M = std::conditional_t<__is_same(T, __bf16), __bf16, float>;  // fp16 goes through fp32 products
  // 64 of c's columns a block where 128 would leave half of the chip without one (577 tokens of 3 heads of 40 x 72, fp32: the outputs 28 us with 128, 22 so)
  const bool few = q.dc <= 64 || static_cast<int64_t>(q.segments) * q.heads * 2 <= device_info().cus;
  if (q.db <= 64) return few ? launch_mix<T, M, 4, 1>(q, st) : launch_mix<T, M, 4, 2>(q, st);
  return few ? launch_mix<T, M, 8, 1>(q, st) : launch_mix<T, M, 8, 2>(q, st);
}

struct Layout {
  size_t spans, carry, copy, bytes;  // copy 0: none needed
};
Layout layout_of(const ppo_decay_attention_args& a) {
  const Plan p = plan_of(a);
  Layout l;
  l.spans = 256;
  l.carry = l.spans + (a.cu_seqlens != nullptr ? static_cast<size_t>(ceil_div(a.tokens * sizeof(Span), 256)) * 256 : 0);
  const size_t states = static_cast<size_t>(a.kv_heads) * a.key_dim * a.value_dim * sizeof(float);
  l.bytes = l.carry + (p.segments - 1) * states;
  l.copy = 0;
  // (query heads of a head may be blocks apart, which read the state that one of them writes)
  const bool forward = a.initial_state != nullptr && a.initial_state == a.final_state, backward = a.d_final_state != nullptr && a.d_final_state == a.d_initial_state;
  if ((forward && (p.segments > 1 || a.q_heads > a.kv_heads)) || (backward && p.segments > 1)) {
    l.copy = static_cast<size_t>(ceil_div(l.bytes, 256)) * 256;
    l.bytes = l.copy + a.sequences * states;
  }
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
  PPO_REQUIRE(n <= 1 || (!backward ? a.out.token_stride : std::max(std::max(a.d_q.token_stride, a.d_k.token_stride), a.d_v.token_stride)) < (int64_t{1} << 31),
              "%s: outputs' tokens lie 2^31 elements apart or more", who);
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

// `from`, `to`: the states (or their gradients) that sequences begin and end with.  What no chunk does for them: sequences without tokens hand theirs on, and
// those that are replaced in place are read from a copy (then `from`), since the block that ends a sequence need not be the only one that begins it.
int prepare(const char* who, const ppo_decay_attention_args& a, const float*& from, float* to, void* workspace, size_t workspace_bytes, hipStream_t st,
            MixArgs& q) {
  const Layout l = layout_of(a);
  PPO_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= l.bytes,
              "%s: workspace too small or not 16-byte aligned (%zu < %zu)", who, workspace_bytes, l.bytes);
  const Plan p = plan_of(a);
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
  const bool in_place = to != nullptr && from == to, handed = to != nullptr && (in_place ? l.copy != 0 : a.cu_seqlens != nullptr || a.tokens == 0);
  SequenceArgs n{a.cu_seqlens, a.cu_type, q.tokens, a.sequences, spans, spans != nullptr ? ceil_div(a.tokens, kInfoThreads) : 0, from, nullptr, 0, in_place};
  if (handed) {
    n.to = in_place ? reinterpret_cast<float*>(base + l.copy) : to;
    n.size = a.kv_heads * q.state_size;
    if (in_place) from = n.to;
  }
  const int64_t blocks = n.token_blocks + (handed ? std::min<int64_t>(a.sequences, 1 << 20) : 0);
  if (blocks == 0) return PPO_OK;
  hipLaunchKernelGGL(decay_sequences_kernel, dim3(static_cast<uint32_t>(blocks)), dim3(kInfoThreads), 0, st, n);
  return check_launch("decay_sequences_kernel");
}

int mix(const ppo_decay_attention_args& a, MixArgs q, hipStream_t st) {
  const int piece = 16 / type_size(a.type);
  if (q.carried == 0) q.ci = q.dc, q.cj = 1;
  else q.ci = 1, q.cj = q.db;  // as the pass before left it, turned over
  q.whole = a.key_dim % piece == 0 && a.value_dim % piece == 0;
  for (const ppo_head_view* v : {&q.a, &q.b, &q.c})  // (rows' offsets within a chunk are products of 24 bits)
    if (v->token_stride * type_size(a.type) >= 1 << 24) q.whole = 0;
  const int64_t row = q.out.token_stride * type_size(a.type), in_row = q.out.head_stride * type_size(a.type);
  q.near = q.whole != 0 && row < 1 << 24 && row % 4 == 0 && in_row % 4 == 0 && reinterpret_cast<uintptr_t>(q.out.data) % 4 == 0;
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
  const float* from = a.initial_state;
  if (int rc = prepare(who, a, from, a.final_state, workspace, workspace_bytes, st, q)) return rc;
  if (a.tokens == 0) return PPO_OK;
  q.a = a.q, q.b = a.k, q.c = a.v, q.out = a.out;
  q.s_in = from, q.s_out = a.final_state, q.cut = a.initial_state != nullptr || a.final_state != nullptr, q.exact = a.final_state != nullptr;
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
  const float* from = a.d_final_state;
  if (int rc = prepare(who, a, from, a.d_initial_state, workspace, workspace_bytes, st, q)) return rc;
  if (a.tokens == 0) return PPO_OK;
  const int group = a.q_heads / a.kv_heads;
  // d_q: in order, S turned over
  q.a = a.out, q.b = a.v, q.c = a.k, q.out = a.d_q;
  q.s_in = a.initial_state, q.cut = a.initial_state != nullptr;
  q.db = a.value_dim, q.dc = a.key_dim, q.si = 1, q.sj = a.value_dim;
  q.ga = group, q.gb = 1, q.w = 1;
  q.x = q.y = static_cast<float>(a.scale), q.z = 1.0f;
  if (int rc = mix(a, q, st)) return rc;
  // d_k, then d_v, whose states are d_k's turned over and which hands on the state's gradient (last: it may lie where d_k's came from): in reverse
  q.reverse = 1, q.w = 0, q.ga = 1, q.gb = group;
  q.x = q.z = static_cast<float>(a.scale), q.y = 1.0f;
  q.s_in = from, q.cut = a.d_final_state != nullptr || a.d_initial_state != nullptr;
  q.exact = a.d_initial_state != nullptr;
  q.a = a.v, q.b = a.out, q.c = a.q, q.out = a.d_k;
  if (int rc = mix(a, q, st)) return rc;
  q.a = a.k, q.b = a.q, q.c = a.out, q.out = a.d_v;
  q.db = a.key_dim, q.dc = a.value_dim, q.si = a.value_dim, q.sj = 1;
  q.s_out = a.d_initial_state, q.carried = 1;
  return mix(a, q, st);
}
