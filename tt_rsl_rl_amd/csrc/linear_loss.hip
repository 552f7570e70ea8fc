// Cross entropy of tokens under a head as wide as the vocabulary, and its gradients, without the logits in memory
// (ppo_linear_log_probs, ppo_linear_cross_entropy).
//
// Rows that count are gathered side by side first, so masked rows cost no products.  Then, with x = hidden weight^T, c = log2(e) /
// temperature, in pieces of the vocabulary:
//   1. products, and of each tile of 256 columns every row's maximum m, S = sum 2^(c (x - m)), E = sum 2^t t (t = c (x - m)) and its
//      token's x; joined over the tiles afterwards: lp = ln2 (c (x_token - m) - log2 S), H = ln2 (log2 S - E / S);
//   2. for the gradient the products again, d = 2^(c (x - m)) / S - [token], rounded to the operands' type, into the workspace both as
//      [rows, columns] and turned; then d_hidden += d weight (fp32 partial sums over pieces and slices of columns, in order) and
//      d_weight = d^T hidden, both times 1 / (N temperature).
// Four products of 2 R V D operations each for three that any way needs: the first one a second time instead of logits kept.
//
// All products are one kernel: out[m, n] = sum_k X[m, k] Y[n, k], both operands with k innermost (what is turned is turned by a copy, a
// few per cent of the products' time), 256 m by 256, 128 or 32 n, eight waves of 32 x 32 x 16 matrix instructions, tiles of 64 k brought
// straight to LDS two deep.  In LDS a row's eight 16-byte pieces change places by the row's number, so that reading a column of pieces
// meets all banks.  An accumulator lane holds one n and rows of m: with the vocabulary along m a row's sums stay in its lane but for one
// shuffle and the waves' join.  fp32 operands are three bf16 parts, and k runs six times over pairs of parts (error 2^-24 and below).
#include "elem.hpp"

namespace ppo {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1000.0f;
constexpr int kGemmThreads = 512;
constexpr int kTileM = 256, kTileK = 64;
constexpr int kRowBytes = kTileK * 2;  // of a tile in LDS
constexpr int kPairs = 6;              // products of fp32 operands' parts
constexpr int kMaxParts = 3;
constexpr int64_t kPieceBytes = int64_t{1} << 28;  // of d in one layout, at most
constexpr int64_t kMinPiece = 2048, kMaxPiece = 32768;

// The operands' 16-bit type: bf16 for fp32's parts.
template <class T>
struct Half {
  typedef T type;
};
template <>
struct Half<float> {
  typedef __bf16 type;
};
template <class T>
constexpr int kParts = sizeof(T) == 4 ? kMaxParts : 1;
// d lies in [-1, 1]; fp16's smallest step near zero would be 6e-8 of that, many tokens' whole probability.
template <class T>
constexpr float kLift = __is_same(T, _Float16) ? 16384.0f : 1.0f;

struct Operand {
  const void* at;     // [part][rows][ld], 16-bit
  int64_t ld, part;   // elements
  int32_t rows;
};

constexpr int kSums = 0, kDiffs = 1, kRowGrad = 2, kWeightGrad = 3;  // what a product is for

struct GemmArgs {
  Operand x, y;          // m, n
  int32_t m, n, steps;   // of 64 k
  const int32_t* count;  // rows that count
  int32_t m_tiles, n_tiles;
  // sums and differences
  int64_t vocab, column0;  // of the piece
  float c;
  const int64_t* token;     // [row]: of the gathered rows
  float *tile_m, *tile_s, *tile_e;  // [tile][sum_rows]
  int64_t sum_rows, tile0;
  float* x_token;
  const float *row_m, *row_inv_s;
  void *d, *d_turned;  // [part][rows][ld_d], [part][columns][ld_t]
  int64_t ld_d, d_part, ld_t, t_part;
  // gradients
  float* partial;  // [slice][rows][m]
  int64_t slice_size;
  int32_t slices, add;
  void* out;  // [n][m]
  int64_t ld_out;
  float denom, inv_temp;
};

template <class M>
__device__ __forceinline__ f32x16 mma(const u32x4& a, const u32x4& b, const f32x16& c) {
  typedef M Frag __attribute__((ext_vector_type(8)));
  if constexpr (__is_same(M, __bf16)) return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(Frag, a), __builtin_bit_cast(Frag, b), c, 0, 0, 0);
  else return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(Frag, a), __builtin_bit_cast(Frag, b), c, 0, 0, 0);
}

// A raw buffer at a wave-uniform address, made of scalar registers (the compiler otherwise may loop over lanes at every load).
__device__ __forceinline__ __amdgpu_buffer_rsrc_t buffer_at(const void* p) {
  const uint64_t a = reinterpret_cast<uint64_t>(p);
  const uint32_t lo = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a)), hi = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(a >> 32));
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(static_cast<uint64_t>(hi) << 32 | lo), 0, 0x7fffffff, 0x00020000);
}

// 16 bytes a lane from offset `off` of a buffer to LDS, at `to` + 16 lane (`to` wave-uniform).
__device__ __forceinline__ void load_to_lds(__amdgpu_buffer_rsrc_t from, uint32_t off, unsigned char* to) {
  __builtin_amdgcn_raw_ptr_buffer_load_lds(from, (__attribute__((address_space(3))) void*)to, 16, off, 0, 0, 0);
}

__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }

// WM x WN waves of TM x TN tiles of 32 x 32.
template <class T, int WM, int WN, int TM, int TN, int JOB>
__global__ __launch_bounds__(kGemmThreads, 1) void linear_gemm_kernel(const GemmArgs q) {
  typedef typename Half<T>::type M;
  constexpr int BN = 32 * TN * WN, BM = 32 * TM * WM, PARTS = kParts<T>;
  static_assert(BM == kTileM && WM * WN * kWave == kGemmThreads);
  constexpr int STAGE = (BM + BN) * kRowBytes;
  constexpr int LOADS_X = BM / 64, LOADS_Y = BN >= 64 ? BN / 64 : 1;  // 1 KB each, per wave
  __shared__ __align__(16) unsigned char lds[2 * STAGE];

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  const int tile = blockIdx.x, mt = tile % q.m_tiles, nt = tile / q.m_tiles;
  const int m0 = mt * BM, n0 = nt * BN;
  const int32_t count = *q.count;
  // (of the last 64 rows the ones past the count are made all the same, as zeros: the second products sum over whole steps)
  if (JOB != kWeightGrad && n0 >= (JOB == kDiffs ? ceil_div(count, kTileK) * kTileK : count)) return;
  int steps = q.steps;
  if (JOB == kWeightGrad) steps = static_cast<int>(ceil_div(count, kTileK));
  int from = 0, to = steps;
  if (JOB == kRowGrad) {  // a slice of k
    const int each = static_cast<int>(ceil_div(steps, q.slices));
    from = min(static_cast<int>(blockIdx.y) * each, steps);
    to = min(from + each, steps);
  }

  // Addresses: a wave's load covers 8 rows of 128 bytes; lane l brings the piece that belongs at its place.
  uint32_t off_x[LOADS_X], off_y[LOADS_Y];
  const auto place = [&](int row) { return static_cast<uint32_t>(((lane % 8) ^ (row / 2 % 8)) * 16); };
#pragma unroll
  for (int i = 0; i < LOADS_X; ++i) {
    const int row = (wave * LOADS_X + i) * 8 + lane / 8;
    off_x[i] = static_cast<uint32_t>(min(m0 + row, q.x.rows - 1) - m0) * static_cast<uint32_t>(q.x.ld * 2) + place(row);
  }
#pragma unroll
  for (int i = 0; i < LOADS_Y; ++i) {
    const int row = (wave * LOADS_Y + i) * 8 + lane / 8;
    off_y[i] = static_cast<uint32_t>(min(n0 + row, q.y.rows - 1) - n0) * static_cast<uint32_t>(q.y.ld * 2) + place(row);
  }
  const char* const base_x = static_cast<const char*>(q.x.at) + static_cast<int64_t>(m0) * q.x.ld * 2;
  const char* const base_y = static_cast<const char*>(q.y.at) + static_cast<int64_t>(n0) * q.y.ld * 2;
  const int per_pair = to - from, total = PARTS == 1 ? per_pair : per_pair * kPairs;
  auto load_stage = [&](int s) {
    int k = s, px = 0, py = 0;
    if constexpr (PARTS > 1) {
      const int pair = s / per_pair;
      k = s - pair * per_pair;
      px = pair == 2 || pair == 3 ? 1 : pair == 5 ? 2 : 0;
      py = pair == 1 || pair == 3 ? 1 : pair == 4 ? 2 : 0;
    }
    const int64_t k_bytes = static_cast<int64_t>(from + k) * kRowBytes;
    const auto rx = buffer_at(base_x + px * q.x.part * 2 + k_bytes), ry = buffer_at(base_y + py * q.y.part * 2 + k_bytes);
    unsigned char* to_lds = lds + (s & 1) * STAGE;
#pragma unroll
    for (int i = 0; i < LOADS_X; ++i) load_to_lds(rx, off_x[i], to_lds + (wave * LOADS_X + i) * 1024);
    if (BN >= 64 || wave < BN / 8)
#pragma unroll
      for (int i = 0; i < LOADS_Y; ++i) load_to_lds(ry, off_y[i], to_lds + BM * kRowBytes + (wave * LOADS_Y + i) * 1024);
  };

  f32x16 acc[TM][TN];
#pragma unroll
  for (int i = 0; i < TM; ++i)
#pragma unroll
    for (int j = 0; j < TN; ++j)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

  const int r32 = lane % 32, half = lane / 32;
  if (total > 0) load_stage(0);
  for (int s = 0; s < total; ++s) {
    wait_loads();
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    if (s + 1 < total) load_stage(s + 1);
    const unsigned char* at = lds + (s & 1) * STAGE;
#pragma unroll
    for (int kk = 0; kk < kTileK / 16; ++kk) {
      u32x4 x[TM], y[TN];
      const int piece = 2 * kk + half;
#pragma unroll
      for (int i = 0; i < TM; ++i) {
        const int row = (wm * TM + i) * 32 + r32;
        x[i] = *reinterpret_cast<const u32x4*>(at + row * kRowBytes + (piece ^ (row / 2 % 8)) * 16);
      }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int row = (wn * TN + j) * 32 + r32;
        y[j] = *reinterpret_cast<const u32x4*>(at + BM * kRowBytes + row * kRowBytes + (piece ^ (row / 2 % 8)) * 16);
      }
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) acc[i][j] = mma<M>(x[i], y[j], acc[i][j]);
    }
  }

  // Element r of acc[i][j]: m = m0 + 32 (wm TM + i) + 8 (r / 4) + 4 half + r % 4,  n = n0 + 32 (wn TN + j) + r32.
  auto m_of = [&](int i, int r) { return 32 * (wm * TM + i) + 8 * (r / 4) + 4 * half + r % 4; };
  if constexpr (JOB == kSums) {
    __syncthreads();
    float* join_at = reinterpret_cast<float*>(lds);  // [WM][3][BN]
    const int64_t left = q.vocab - q.column0 - m0;   // columns of the tile that are there
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 32 * (wn * TN + j) + r32;
      const int64_t tok = n < count ? q.token[n] - q.column0 - m0 : -1;
      float m = -INFINITY;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int col = m_of(i, r);
          if (col >= left) acc[i][j][r] = -INFINITY;
          if (col == tok) q.x_token[n] = acc[i][j][r];
          m = fmaxf(m, acc[i][j][r]);
        }
      m = fmaxf(m, __shfl_xor(m, 32, kWave));
      const float zero = m > -INFINITY ? m : 0.0f;
      float s = 0.0f, e = 0.0f;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const float t = (acc[i][j][r] - zero) * q.c, p = __builtin_amdgcn_exp2f(t);
          s += p;
          e = fmaf(p, fmaxf(t, kFloor), e);
        }
      s += __shfl_xor(s, 32, kWave);
      e += __shfl_xor(e, 32, kWave);
      if (half == 0) {
        const int b = 32 * (wn * TN + j) + r32;
        join_at[(wm * 3 + 0) * BN + b] = m;
        join_at[(wm * 3 + 1) * BN + b] = s;
        join_at[(wm * 3 + 2) * BN + b] = e;
      }
    }
    __syncthreads();
    for (int b = threadIdx.x; b < BN; b += kGemmThreads) {
      if (n0 + b >= count) continue;
      float m = -INFINITY, s = 0.0f, e = 0.0f;
#pragma unroll
      for (int w = 0; w < WM; ++w) m = fmaxf(m, join_at[(w * 3) * BN + b]);
#pragma unroll
      for (int w = 0; w < WM; ++w) {
        const float mw = join_at[(w * 3) * BN + b], sw = join_at[(w * 3 + 1) * BN + b], ew = join_at[(w * 3 + 2) * BN + b];
        const float t = mw == m ? 0.0f : fmaxf((mw - m) * q.c, kFloor), f = __builtin_amdgcn_exp2f(t);
        s = fmaf(sw, f, s);
        e = fmaf(ew + sw * t, f, e);
      }
      const int64_t at = (q.tile0 + mt) * q.sum_rows + n0 + b;
      q.tile_m[at] = m, q.tile_s[at] = s, q.tile_e[at] = e;
    }
  } else if constexpr (JOB == kDiffs) {
    const int64_t left = q.vocab - q.column0 - m0;
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 32 * (wn * TN + j) + r32;
      const bool live = n < count;
      const int64_t tok = live ? q.token[n] - q.column0 - m0 : -1;
      const float m = live ? q.row_m[n] : 0.0f, inv = live ? q.row_inv_s[n] : 0.0f;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          float v[4];
          const int col = m_of(i, 4 * r4);
#pragma unroll
          for (int r = 0; r < 4; ++r) {
            const float p = __builtin_amdgcn_exp2f((acc[i][j][4 * r4 + r] - m) * q.c) * inv;
            v[r] = live && col + r < left ? (p - (col + r == tok ? 1.0f : 0.0f)) * kLift<T> : 0.0f;
          }
#pragma unroll
          for (int part = 0; part < PARTS; ++part) {
            typedef M Four __attribute__((ext_vector_type(4)));
            Four f;
#pragma unroll
            for (int r = 0; r < 4; ++r) {
              f[r] = static_cast<M>(v[r]);
              v[r] -= static_cast<float>(f[r]);
            }
            // (rows of a tile past the gathered ones are there too, as zeros, in both layouts; columns up to the tile's end as well)
            if (q.d != nullptr && n < q.n) *reinterpret_cast<Four*>(static_cast<M*>(q.d) + part * q.d_part + static_cast<int64_t>(n) * q.ld_d + m0 + col) = f;
            if (q.d_turned != nullptr && n < q.n)
#pragma unroll
              for (int r = 0; r < 4; ++r) (static_cast<M*>(q.d_turned) + part * q.t_part)[static_cast<int64_t>(m0 + col + r) * q.ld_t + n] = f[r];
          }
        }
    }
  } else {
    const float factor = 1.0f / kLift<T> * (JOB == kWeightGrad ? q.inv_temp / (q.denom > 0.0f ? q.denom : static_cast<float>(max(count, 1))) : 1.0f);
#pragma unroll
    for (int j = 0; j < TN; ++j) {
      const int n = n0 + 32 * (wn * TN + j) + r32;
      if (n >= q.n) continue;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
          const int m = m0 + m_of(i, 4 * r4);
          if constexpr (JOB == kRowGrad) {
            float* at = q.partial + blockIdx.y * q.slice_size + static_cast<int64_t>(n) * q.m + m;
#pragma unroll
            for (int r = 0; r < 4; ++r)
              if (m + r < q.m) at[r] = q.add != 0 ? at[r] + acc[i][j][4 * r4 + r] * factor : acc[i][j][4 * r4 + r] * factor;
          } else {
            T* at = static_cast<T*>(q.out) + static_cast<int64_t>(n) * q.ld_out + m;
            if (m + 4 <= q.m) {
              typedef T Four __attribute__((ext_vector_type(4), aligned(sizeof(T))));
              Four f;
#pragma unroll
              for (int r = 0; r < 4; ++r) f[r] = static_cast<T>(acc[i][j][4 * r4 + r] * factor);
              *reinterpret_cast<Four*>(at) = f;
            } else {
#pragma unroll
              for (int r = 0; r < 4; ++r)
                if (m + r < q.m) at[r] = static_cast<T>(acc[i][j][4 * r4 + r] * factor);
            }
          }
        }
    }
  }
}

// ---- the rows that count ----

constexpr int kRowThreads = 1024;
struct RowArgs {
  ppo_linear_loss_args a;
  int32_t* count;
  int32_t* source;   // [gathered row]: its row
  int32_t* gathered; // [row]: its gathered row, or -1
  int64_t* token;    // [gathered row]
  float *tile_m, *tile_s, *tile_e;
  int64_t sum_rows, tiles;
  float* x_token;
  float *row_m, *row_inv_s, *row_lp, *row_h;
  const float* partial;
  int64_t slice_size;
  int32_t slices;
  float c;
};

// One block: the rows that count, in order.
__global__ __launch_bounds__(kRowThreads) void linear_rows_kernel(const RowArgs q) {
  __shared__ int32_t waves[kRowThreads / kWave + 1];
  int32_t before = 0;
  for (int64_t r0 = 0; r0 < q.a.rows; r0 += kRowThreads) {
    const int64_t r = r0 + threadIdx.x;
    int64_t tok = -1;
    if (r < q.a.rows && (q.a.mask == nullptr || q.a.mask[r] != 0)) tok = token_at(q.a.tokens, q.a.token_type, r, q.a.vocab);
    const uint64_t in = __ballot(tok >= 0);
    const int lane = threadIdx.x % kWave, wave = threadIdx.x / kWave;
    if (lane == 0) waves[wave] = __popcll(in);
    __syncthreads();
    int32_t at = before, all = 0;
    for (int w = 0; w < kRowThreads / kWave; ++w) {
      if (w < wave) at += waves[w];
      all += waves[w];
    }
    at += __popcll(in & ((uint64_t{1} << lane) - 1));
    if (r < q.a.rows) q.gathered[r] = tok >= 0 ? at : -1;
    if (tok >= 0) q.source[at] = static_cast<int32_t>(r), q.token[at] = tok;
    before += all;
    __syncthreads();
  }
  if (threadIdx.x == 0) *q.count = before;
}

// ---- operands: rows as 16-bit parts, padded with zeros along k; and turned ----

struct PackArgs {
  const void* src;
  int64_t ld, rows, dim;     // rows there, of dim elements
  const int32_t* source;     // gathered rows, and how many
  const int32_t* count;
  void* dst;                 // [part][out_rows][ld_dst]
  int64_t ld_dst, part, out_rows;
};

template <class T, class M>
__device__ __forceinline__ void store_parts(M* at, int64_t part, float x) {
#pragma unroll
  for (int p = 0; p < kParts<T>; ++p) {
    const M h = static_cast<M>(x);
    at[p * part] = h;
    x -= static_cast<float>(h);
  }
}

constexpr int kPackThreads = 256;
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_pack_kernel(const PackArgs q) {
  typedef typename Half<T>::type M;
  const int64_t row = blockIdx.x;
  const int64_t rows = q.count != nullptr ? static_cast<int64_t>(*q.count) : q.rows;
  const T* from = nullptr;
  if (row < rows) from = static_cast<const T*>(q.src) + (q.source != nullptr ? q.source[row] : row) * q.ld;
  M* to = static_cast<M*>(q.dst) + row * q.ld_dst;
  for (int64_t k = threadIdx.x; k < q.ld_dst; k += kPackThreads)
    store_parts<T>(to + k, q.part, from != nullptr && k < q.dim ? static_cast<float>(from[k]) : 0.0f);
}

// dst[k][row]: 64 x 64 tiles through LDS.
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_turn_kernel(const PackArgs q) {
  typedef typename Half<T>::type M;
  __shared__ float tile[64][65];
  const int64_t rows = q.count != nullptr ? static_cast<int64_t>(*q.count) : q.rows;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 64, k0 = static_cast<int64_t>(blockIdx.y) * 64;
  const int lane = threadIdx.x % 64, part = threadIdx.x / 64;
  for (int i = part; i < 64; i += 4) {
    const int64_t row = row0 + i, k = k0 + lane;
    float x = 0.0f;
    if (row < rows && k < q.dim) x = static_cast<float>((static_cast<const T*>(q.src) + (q.source != nullptr ? q.source[row] : row) * q.ld)[k]);
    tile[i][lane] = x;
  }
  __syncthreads();
  for (int i = part; i < 64; i += 4) {
    const int64_t k = k0 + i;
    if (k < q.dim) store_parts<T>(static_cast<M*>(q.dst) + k * q.ld_dst + row0 + lane, q.part, tile[lane][i]);
  }
}

// ---- rows: the tiles' sums joined, log-probabilities, the loss ----

constexpr int kJoinThreads = 256;
__global__ __launch_bounds__(kJoinThreads) void linear_join_kernel(const RowArgs q) {
  const int lane = threadIdx.x % kWave;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * (kJoinThreads / kWave) + threadIdx.x / kWave;
  if (n >= *q.count) return;
  float m = -INFINITY;
  for (int64_t t = lane; t < q.tiles; t += kWave) m = fmaxf(m, q.tile_m[t * q.sum_rows + n]);
  for (int d = kWave / 2; d > 0; d >>= 1) m = fmaxf(m, __shfl_xor(m, d, kWave));
  float s = 0.0f, e = 0.0f;
  for (int64_t t = lane; t < q.tiles; t += kWave) {
    const float mt = q.tile_m[t * q.sum_rows + n], st = q.tile_s[t * q.sum_rows + n], et = q.tile_e[t * q.sum_rows + n];
    const float u = mt == m ? 0.0f : fmaxf((mt - m) * q.c, kFloor), f = __builtin_amdgcn_exp2f(u);
    s = fmaf(st, f, s);
    e = fmaf(et + st * u, f, e);
  }
  for (int d = kWave / 2; d > 0; d >>= 1) s += __shfl_xor(s, d, kWave), e += __shfl_xor(e, d, kWave);
  if (lane != 0) return;
  const float log2_s = log2f(s), lp = kLn2 * ((q.x_token[n] - m) * q.c - log2_s), h = kLn2 * (log2_s - e / s);
  q.row_m[n] = m, q.row_inv_s[n] = 1.0f / s, q.row_lp[n] = lp, q.row_h[n] = h;
}

__global__ __launch_bounds__(kJoinThreads) void linear_scatter_kernel(const RowArgs q) {
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kJoinThreads + threadIdx.x;
  if (r >= q.a.rows) return;
  const int32_t n = q.gathered[r];
  if (q.a.logp != nullptr) q.a.logp[r] = n >= 0 ? q.row_lp[n] : 0.0f;
  if (q.a.entropy != nullptr) q.a.entropy[r] = n >= 0 ? q.row_h[n] : 0.0f;
}

__global__ __launch_bounds__(kRowThreads) void linear_stats_kernel(const RowArgs q) {
  __shared__ double part[2][kRowThreads / kWave];
  const int32_t count = *q.count;
  double lp = 0.0, h = 0.0;
  for (int32_t n = threadIdx.x; n < count; n += kRowThreads) lp += static_cast<double>(q.row_lp[n]), h += static_cast<double>(q.row_h[n]);
  for (int d = kWave / 2; d > 0; d >>= 1) lp += __shfl_xor(lp, d, kWave), h += __shfl_xor(h, d, kWave);
  if (threadIdx.x % kWave == 0) part[0][threadIdx.x / kWave] = lp, part[1][threadIdx.x / kWave] = h;
  __syncthreads();
  if (threadIdx.x != 0) return;
  lp = h = 0.0;
  for (int w = 0; w < kRowThreads / kWave; ++w) lp += part[0][w], h += part[1][w];
  const double n = q.a.denom > 0.0 ? q.a.denom : static_cast<double>(count);
  q.a.stats[0] = count > 0 ? static_cast<float>(-lp / n) : 0.0f;
  q.a.stats[1] = count > 0 ? static_cast<float>(h / n) : 0.0f;
  q.a.stats[2] = static_cast<float>(n);
  q.a.stats[3] = 0.0f;
}

// d_hidden: the slices' sums of each row, zeros where a row does not count.
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_row_grad_kernel(const RowArgs q) {
  const int64_t r = blockIdx.x;
  const int32_t n = q.gathered[r];
  T* to = static_cast<T*>(q.a.d_hidden) + r * q.a.ld_d_hidden;
  const float factor = static_cast<float>(1.0 / (q.a.temperature * (q.a.denom > 0.0 ? q.a.denom : static_cast<double>(max(*q.count, 1)))));
  for (int64_t k = threadIdx.x; k < q.a.dim; k += kPackThreads) {
    float x = 0.0f;
    if (n >= 0)
      for (int s = 0; s < q.slices; ++s) x += q.partial[s * q.slice_size + n * q.a.dim + k];
    to[k] = static_cast<T>(x * factor);
  }
}

// ---- the host's part ----

struct Plan {
  int64_t rows, k, piece, pieces;  // rows and k padded to whole tiles of k
  int parts, slices, n_tile;
  bool direct;  // the weight is an operand as it lies
  size_t count, source, gathered, token, sums, x_token, row, hidden, hidden_turned, weight, weight_turned, d, d_turned, partial, bytes;
};

int64_t up(int64_t x, int64_t to) { return ceil_div(x, to) * to; }

Plan plan_of(const ppo_linear_loss_args& a, bool gradient) {
  Plan p{};
  p.parts = a.type == PPO_TYPE_F32 ? kMaxParts : 1;
  p.rows = up(std::max<int64_t>(a.rows, 1), kTileK);
  p.k = up(a.dim, kTileK);
  p.direct = a.type != PPO_TYPE_F32 && a.dim % kTileK == 0 && a.ld_weight % 8 == 0 && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
  // columns at a time: d of a piece up to kPieceBytes
  int64_t piece = kPieceBytes / (p.rows * 2 * p.parts) / kTileM * kTileM;
  piece = std::min(std::max(piece, kMinPiece), kMaxPiece);
  if (!gradient && p.direct) piece = up(a.vocab, kTileM);
  p.piece = std::min(piece, up(a.vocab, kTileM));
  p.pieces = ceil_div(a.vocab, p.piece);
  p.n_tile = a.rows <= 32 ? 32 : a.rows <= 128 || (a.rows > 256 && a.rows <= 384) ? 128 : 256;
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  const int64_t tiles = ceil_div(a.dim, kTileM) * ceil_div(a.rows, p.n_tile), steps = p.piece / kTileK;
  p.slices = static_cast<int>(std::max<int64_t>(1, std::min(cus / std::max<int64_t>(tiles, 1), steps / 8)));
  size_t at = 256;
  auto room = [&](size_t n) {
    const size_t from = at;
    at += up(n, 256);
    return from;
  };
  p.count = 0;
  p.source = room(p.rows * 4);
  p.gathered = room(p.rows * 4);
  p.token = room(p.rows * 8);
  p.sums = room(3 * ceil_div(a.vocab, kTileM) * p.rows * 4);
  p.x_token = room(p.rows * 4);
  p.row = room(4 * p.rows * 4);
  p.hidden = room(p.parts * p.rows * p.k * 2);
  p.weight = room(p.direct ? 0 : p.parts * p.piece * p.k * 2);
  if (gradient) {
    if (a.d_hidden != nullptr) {
      p.weight_turned = room(p.parts * a.dim * p.piece * 2);
      p.d = room(p.parts * p.rows * p.piece * 2);
      p.partial = room(static_cast<size_t>(p.slices) * p.rows * a.dim * 4);
    }
    if (a.d_weight != nullptr) {
      p.hidden_turned = room(p.parts * a.dim * p.rows * 2);
      p.d_turned = room(p.parts * p.piece * p.rows * 2);
    }
  }
  p.bytes = at;
  return p;
}

template <class T, int JOB>
int launch_gemm(GemmArgs g, int n_tile, hipStream_t st) {
  if (JOB == kWeightGrad) n_tile = 256;  // n is the vocabulary there
  g.m_tiles = static_cast<int32_t>(ceil_div(g.m, kTileM));
  g.n_tiles = static_cast<int32_t>(ceil_div(g.n, n_tile));
  const dim3 grid(static_cast<uint32_t>(g.m_tiles) * static_cast<uint32_t>(g.n_tiles), JOB == kRowGrad ? g.slices : 1);
  if (n_tile == 256) hipLaunchKernelGGL((linear_gemm_kernel<T, 2, 4, 4, 2, JOB>), grid, dim3(kGemmThreads), 0, st, g);
  else if constexpr (JOB != kWeightGrad) {
    if (n_tile == 128) hipLaunchKernelGGL((linear_gemm_kernel<T, 4, 2, 2, 2, JOB>), grid, dim3(kGemmThreads), 0, st, g);
    else hipLaunchKernelGGL((linear_gemm_kernel<T, 8, 1, 1, 1, JOB>), grid, dim3(kGemmThreads), 0, st, g);
  }
  return check_launch("linear_gemm_kernel");
}

template <class T>
int run_typed(const ppo_linear_loss_args& a, const Plan& p, char* ws, hipStream_t st, bool gradient) {
  const int64_t size = sizeof(T);
  RowArgs r{};
  r.a = a;
  r.count = reinterpret_cast<int32_t*>(ws + p.count);
  r.source = reinterpret_cast<int32_t*>(ws + p.source);
  r.gathered = reinterpret_cast<int32_t*>(ws + p.gathered);
  r.token = reinterpret_cast<int64_t*>(ws + p.token);
  r.sum_rows = p.rows;
  r.tiles = ceil_div(a.vocab, kTileM);
  r.tile_m = reinterpret_cast<float*>(ws + p.sums);
  r.tile_s = r.tile_m + r.tiles * p.rows;
  r.tile_e = r.tile_s + r.tiles * p.rows;
  r.x_token = reinterpret_cast<float*>(ws + p.x_token);
  r.row_m = reinterpret_cast<float*>(ws + p.row);
  r.row_inv_s = r.row_m + p.rows;
  r.row_lp = r.row_inv_s + p.rows;
  r.row_h = r.row_lp + p.rows;
  r.c = static_cast<float>(1.4426950408889634 / a.temperature);
  r.partial = reinterpret_cast<const float*>(ws + p.partial);
  r.slice_size = p.rows * a.dim;
  r.slices = p.slices;
  hipLaunchKernelGGL(linear_rows_kernel, dim3(1), dim3(kRowThreads), 0, st, r);
  if (int rc = check_launch("linear_rows_kernel")) return rc;

  PackArgs h{a.hidden, a.ld_hidden, a.rows, a.dim, r.source, r.count, ws + p.hidden, p.k, p.rows * p.k, p.rows};
  hipLaunchKernelGGL(linear_pack_kernel<T>, dim3(static_cast<uint32_t>(p.rows)), dim3(kPackThreads), 0, st, h);
  if (int rc = check_launch("linear_pack_kernel")) return rc;
  const bool to_hidden = gradient && a.d_hidden != nullptr, to_weight = gradient && a.d_weight != nullptr;
  if (to_weight) {
    h.dst = ws + p.hidden_turned, h.ld_dst = p.rows, h.part = a.dim * p.rows;
    hipLaunchKernelGGL(linear_turn_kernel<T>, dim3(static_cast<uint32_t>(p.rows / 64), static_cast<uint32_t>(ceil_div(a.dim, 64))), dim3(kPackThreads), 0, st, h);
    if (int rc = check_launch("linear_turn_kernel")) return rc;
  }

  GemmArgs g{};
  g.y = Operand{ws + p.hidden, p.k, p.rows * p.k, static_cast<int32_t>(p.rows)};
  g.n = static_cast<int32_t>(p.rows);
  g.steps = static_cast<int32_t>(p.k / kTileK);
  g.count = r.count;
  g.vocab = a.vocab;
  g.c = r.c;
  g.token = r.token;
  g.tile_m = r.tile_m, g.tile_s = r.tile_s, g.tile_e = r.tile_e, g.sum_rows = r.sum_rows;
  g.x_token = r.x_token;
  g.row_m = r.row_m, g.row_inv_s = r.row_inv_s;
  g.denom = static_cast<float>(a.denom);
  g.inv_temp = static_cast<float>(1.0 / a.temperature);
  auto weight_piece = [&](int64_t v0, int64_t n) -> int {
    const char* from = static_cast<const char*>(a.weight) + v0 * a.ld_weight * size;
    g.m = static_cast<int32_t>(n);
    g.column0 = v0;
    if (p.direct) {
      g.x = Operand{from, a.ld_weight, 0, static_cast<int32_t>(n)};
      return PPO_OK;
    }
    const PackArgs w{from, a.ld_weight, n, a.dim, nullptr, nullptr, ws + p.weight, p.k, p.piece * p.k, n};
    hipLaunchKernelGGL(linear_pack_kernel<T>, dim3(static_cast<uint32_t>(n)), dim3(kPackThreads), 0, st, w);
    g.x = Operand{ws + p.weight, p.k, p.piece * p.k, static_cast<int32_t>(n)};
    return check_launch("linear_pack_kernel");
  };
  for (int64_t v0 = 0; v0 < a.vocab && a.rows > 0; v0 += p.piece) {
    if (int rc = weight_piece(v0, std::min(p.piece, a.vocab - v0))) return rc;
    g.tile0 = v0 / kTileM;
    if (int rc = launch_gemm<T, kSums>(g, p.n_tile, st)) return rc;
  }
  if (a.rows > 0) {
    hipLaunchKernelGGL(linear_join_kernel, dim3(static_cast<uint32_t>(ceil_div(a.rows, kJoinThreads / kWave))), dim3(kJoinThreads), 0, st, r);
    if (int rc = check_launch("linear_join_kernel")) return rc;
    if (a.logp != nullptr || a.entropy != nullptr) {
      hipLaunchKernelGGL(linear_scatter_kernel, dim3(static_cast<uint32_t>(ceil_div(a.rows, kJoinThreads))), dim3(kJoinThreads), 0, st, r);
      if (int rc = check_launch("linear_scatter_kernel")) return rc;
    }
  }
  if (!gradient) return PPO_OK;
  hipLaunchKernelGGL(linear_stats_kernel, dim3(1), dim3(kRowThreads), 0, st, r);
  if (int rc = check_launch("linear_stats_kernel")) return rc;
  if (!to_hidden && !to_weight) return PPO_OK;

  for (int64_t v0 = 0; v0 < a.vocab; v0 += p.piece) {
    const int64_t n = std::min(p.piece, a.vocab - v0);
    if (p.pieces > 1 || v0 == 0) {
      if (p.pieces > 1 || p.direct) {
        if (int rc = weight_piece(v0, n)) return rc;
      }
    }
    const Operand hidden = g.y, weight = g.x;
    g.d = to_hidden ? ws + p.d : nullptr;
    g.d_turned = to_weight ? ws + p.d_turned : nullptr;
    g.ld_d = p.piece, g.d_part = p.rows * p.piece;
    g.ld_t = p.rows, g.t_part = p.piece * p.rows;
    if (a.rows > 0)
      if (int rc = launch_gemm<T, kDiffs>(g, p.n_tile, st)) return rc;
    if (to_hidden && a.rows > 0) {
      const PackArgs w{static_cast<const char*>(a.weight) + v0 * a.ld_weight * size, a.ld_weight, n, a.dim, nullptr, nullptr, ws + p.weight_turned, p.piece,
                       a.dim * p.piece, 0};
      hipLaunchKernelGGL(linear_turn_kernel<T>, dim3(static_cast<uint32_t>(ceil_div(n, 64)), static_cast<uint32_t>(ceil_div(a.dim, 64))), dim3(kPackThreads), 0, st,
                         w);
      if (int rc = check_launch("linear_turn_kernel")) return rc;
      GemmArgs b = g;
      b.x = Operand{ws + p.weight_turned, p.piece, a.dim * p.piece, static_cast<int32_t>(a.dim)};
      b.y = Operand{ws + p.d, p.piece, p.rows * p.piece, static_cast<int32_t>(p.rows)};
      b.m = static_cast<int32_t>(a.dim);
      b.steps = static_cast<int32_t>(ceil_div(n, kTileK));
      b.partial = reinterpret_cast<float*>(ws + p.partial);
      b.slice_size = r.slice_size;
      b.slices = p.slices;
      b.add = v0 > 0;
      if (int rc = launch_gemm<T, kRowGrad>(b, p.n_tile, st)) return rc;
    }
    if (to_weight) {
      GemmArgs b = g;
      b.x = Operand{ws + p.hidden_turned, p.rows, a.dim * p.rows, static_cast<int32_t>(a.dim)};
      b.y = Operand{ws + p.d_turned, p.rows, p.piece * p.rows, static_cast<int32_t>(n)};
      b.m = static_cast<int32_t>(a.dim);
      b.n = static_cast<int32_t>(n);
      b.out = static_cast<char*>(a.d_weight) + v0 * a.ld_d_weight * size;
      b.ld_out = a.ld_d_weight;
      if (int rc = launch_gemm<T, kWeightGrad>(b, p.n_tile, st)) return rc;
    }
    g.x = weight, g.y = hidden;
  }
  if (to_hidden && a.rows > 0) {
    hipLaunchKernelGGL(linear_row_grad_kernel<T>, dim3(static_cast<uint32_t>(a.rows)), dim3(kPackThreads), 0, st, r);
    return check_launch("linear_row_grad_kernel");
  }
  return PPO_OK;
}

constexpr int64_t kMostRows = int64_t{1} << 22, kMostDim = int64_t{1} << 20;  // so that a tile's offsets stay in 31 bits
bool sizes_ok(const ppo_linear_loss_args& a) {
  return a.rows >= 0 && a.rows < kMostRows && a.vocab >= 1 && a.vocab < (int64_t{1} << 30) && a.dim >= 1 && a.dim <= kMostDim && type_ok(a.type);
}

int check(const char* who, const ppo_linear_loss_args* args, bool gradient) {
  PPO_REQUIRE(args != nullptr, "%s: null arguments", who);
  const ppo_linear_loss_args& a = *args;
  PPO_REQUIRE(type_ok(a.type), "%s: type=%d", who, a.type);
  PPO_REQUIRE(sizes_ok(a), "%s: rows=%lld vocab=%lld dim=%lld", who, (long long)a.rows, (long long)a.vocab, (long long)a.dim);
  PPO_REQUIRE(a.token_type == PPO_TOKENS_I64 || a.token_type == PPO_TOKENS_I32, "%s: token_type=%d", who, a.token_type);
  PPO_REQUIRE(a.temperature >= 1e-6 && a.temperature <= 1e6, "%s: temperature=%g", who, a.temperature);
  const int64_t ld_most = int64_t{1} << 21;
  PPO_REQUIRE(a.ld_hidden >= a.dim && a.ld_weight >= a.dim && (a.d_hidden == nullptr || !gradient || a.ld_d_hidden >= a.dim) &&
                  (a.d_weight == nullptr || !gradient || a.ld_d_weight >= a.dim),
              "%s: leading dimensions below dim=%lld", who, (long long)a.dim);
  PPO_REQUIRE(a.ld_weight <= ld_most, "%s: ld_weight=%lld", who, (long long)a.ld_weight);
  PPO_REQUIRE(a.weight != nullptr && (a.rows == 0 || (a.hidden != nullptr && a.tokens != nullptr)), "%s: null pointer", who);
  const int64_t size = type_size(a.type);
  PPO_REQUIRE(reinterpret_cast<uintptr_t>(a.hidden) % size == 0 && reinterpret_cast<uintptr_t>(a.weight) % size == 0 &&
                  reinterpret_cast<uintptr_t>(a.d_hidden) % size == 0 && reinterpret_cast<uintptr_t>(a.d_weight) % size == 0 &&
                  reinterpret_cast<uintptr_t>(a.tokens) % (a.token_type == PPO_TOKENS_I64 ? 8 : 4) == 0,
              "%s: pointers must be aligned to their elements", who);
  if (gradient) {
    PPO_REQUIRE(a.stats != nullptr, "%s: null pointer", who);
    PPO_REQUIRE(a.denom >= 0.0 && a.denom < 1e30, "%s: denom=%g", who, a.denom);
  }
  const int64_t n = a.rows;
  const Rows none{nullptr, 0, 0, 0};
  const Rows in[] = {n > 0 ? Rows{a.hidden, n, a.dim * size, a.ld_hidden * size} : none, Rows{a.weight, a.vocab, a.dim * size, a.ld_weight * size},
                     n > 0 ? vector_of(a.tokens, n * (a.token_type == PPO_TOKENS_I64 ? 8 : 4)) : none, n > 0 ? vector_of(a.mask, n) : none};
  const Rows out[] = {n > 0 ? vector_of(a.logp, n * 4) : none, n > 0 ? vector_of(a.entropy, n * 4) : none, gradient ? vector_of(a.stats, 16) : none,
                      gradient && n > 0 ? Rows{a.d_hidden, n, a.dim * size, a.ld_d_hidden * size} : none,
                      gradient ? Rows{a.d_weight, a.vocab, a.dim * size, a.ld_d_weight * size} : none};
  for (int i = 0; i < 5; ++i) {
    for (const Rows& x : in) PPO_REQUIRE(!overlap(out[i], x), "%s: an output overlaps an input", who);
    for (int k = 0; k < i; ++k) PPO_REQUIRE(!overlap(out[i], out[k]), "%s: outputs overlap", who);
  }
  return PPO_OK;
}

int run(const char* who, const ppo_linear_loss_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream, bool gradient) {
  if (int rc = check(who, args, gradient)) return rc;
  const ppo_linear_loss_args& a = *args;
  if (!gradient && (a.rows == 0 || (a.logp == nullptr && a.entropy == nullptr))) return PPO_OK;
  const Plan p = plan_of(a, gradient);
  PPO_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 16 == 0 && workspace_bytes >= p.bytes,
              "%s: workspace too small or not 16-byte aligned (%zu < %zu)", who, workspace_bytes, p.bytes);
  int rc = PPO_OK;
  with_type(a.type, [&](auto t) { rc = run_typed<decltype(t)>(a, p, static_cast<char*>(workspace), static_cast<hipStream_t>(stream), gradient); });
  return rc;
}

}  // namespace
}  // namespace ppo

using namespace ppo;

extern "C" size_t ppo_linear_loss_workspace_bytes(const ppo_linear_loss_args* args, int32_t gradient) {
  return args != nullptr && sizes_ok(*args) ? plan_of(*args, gradient != 0).bytes : 0;
}

extern "C" int ppo_linear_log_probs(const ppo_linear_loss_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream) {
  return run("ppo_linear_log_probs", args, workspace, workspace_bytes, stream, false);
}

extern "C" int ppo_linear_cross_entropy(const ppo_linear_loss_args* args, void* workspace, size_t workspace_bytes, ppo_stream_t stream) {
  return run("ppo_linear_cross_entropy", args, workspace, workspace_bytes, stream, true);
}
