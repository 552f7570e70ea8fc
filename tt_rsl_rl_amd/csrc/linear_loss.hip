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
// few per cent of the products' time), 256 m by 256, 128 or 32 n, eight waves of 32 x 32 x 16 matrix instructions, tiles of 64 (32) k brought
// straight to LDS, two to four deep.  In LDS a row's 16-byte pieces change places by the row's number, so that reading a column of pieces
// meets all banks.  An accumulator lane holds one n and rows of m: with the vocabulary along m a row's sums stay in its lane but for one
// shuffle and the waves' join.  fp32 operands are three bf16 parts, six products of which are taken (what is left out is 2^-24 and below).
//
// Bound by the matrix cores.  8,192 rows, of which 6,144 count, of 2,048 over 131,072 columns, bf16, for each 16,384 columns (412 GFLOP a product): sums 379 us,
// differences 431, d_hidden 394, d_weight 329 (1,250 TFLOP/s), turning the weight 28 (134 MB in and out, 4.8 TB/s).
#include <numeric>

#include "elem.hpp"

namespace ppo {
namespace {

typedef float f32x16 __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr float kLn2 = 0.69314718055994530942f;
constexpr float kFloor = -1000.0f;
constexpr int kGemmThreads = 512;
constexpr int kTileM = 256, kTileK = 64;  // (operands' k is padded to whole tiles of 64)
constexpr int kMaxParts = 3;
// A piece's columns: d in both layouts and the weight's copies take up to so much (a piece more costs a reading and a writing of d_hidden's sums).
constexpr int64_t kPieceBytes = int64_t{3} << 28;
constexpr int64_t kMinPiece = 2048;
constexpr int64_t kMostTiles = int64_t{1} << 22;  // of a product: a launch holds fewer than 2^32 threads
constexpr int64_t kKeptBytes = int64_t{1} << 28;

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
template <class T>
constexpr int kStep = sizeof(T) == 4 ? 32 : 64;  // k of a stage (bf16: 32, four stages deep, took 6 to 9 % longer)
// d lies in [-1, 1]; fp16's smallest step near zero would be 6e-8 of that, many tokens' whole probability.
template <class T>
constexpr float kLift = __is_same(T, _Float16) ? 16384.0f : 1.0f;

// How d_hidden's tiles are shared out to the compute units; only the device knows how many rows count.  Tiles that make whole rounds take one block each.  Of the
// rest, few are cut into slices of k, as many as fill one round; many leave a part of their k, 1 / (per + 1), to the units that would idle, `per` tiles to each
// of these.  Every share of a tile has its own sums, the first ones tile after tile, the others behind them.  (192 tiles on 256 units, 16,384 columns: 482 us a tile
// each, so 400; 6 tiles of 193 rows by 515, fp32, 50,021 columns: 155 us in two rounds of slices, 123 in one.)
struct Shares {
  int whole, rest, slots, per;  // per 0: slices
};
__device__ __forceinline__ Shares shares_of(int tiles, int cus, int steps) {
  Shares s{tiles / cus * cus, 0, 1, 0};
  s.rest = tiles - s.whole;
  if (s.rest == 0) return s;
  if (2 * s.rest <= cus) {
    s.slots = min(cus / s.rest, max(steps / 8, 1));
  } else {
    const int per = static_cast<int>(ceil_div(s.rest, cus - s.rest));
    if (per <= 8) s.slots = 2, s.per = per;
  }
  return s;
}

struct Operand {
  const void* at;     // [part][rows][ld], 16-bit
  int64_t ld, part;   // elements
  int32_t rows;
};

constexpr int kSums = 0, kDiffs = 1, kRowGrad = 2, kWeightGrad = 3;  // what a product is for

struct GemmArgs {
  Operand x, y;          // m, n
  int32_t m, n, steps;   // of the kernel's STEP k
  const int32_t* count;  // rows that count
  int32_t m_tiles, n_tiles, xcds;
  // sums and differences
  int64_t vocab, column0;  // of the piece
  float c;
  const int64_t* token;     // [row]: of the gathered rows
  float *tile_m, *tile_s, *tile_e;  // [tile][sum_rows]
  int64_t sum_rows, tile0;
  float* x_token;
  const float *row_m, *row_inv_s;
  float* kept;  // [row][ld_kept]: the products themselves, NULL: not kept
  int64_t ld_kept;
  void *d, *d_turned;  // [part][rows][ld_d], [part][columns][ld_t]
  int64_t ld_d, d_part, ld_t, t_part;
  // gradients
  float* partial;  // [slice][rows][m]
  int32_t cus, all_steps, add;  // all_steps: of a whole piece, which decides the slices
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

// All but the wave's last N loads have arrived.
template <int N>
__device__ __forceinline__ void wait_loads() { asm volatile("s_waitcnt vmcnt(%0)" ::"n"(N) : "memory"); }

// WM x WN waves of TM x TN tiles of 32 x 32.
template <class T, int WM, int WN, int TM, int TN, int JOB>
__global__ __launch_bounds__(kGemmThreads, 1) void linear_gemm_kernel(const GemmArgs q) {
  typedef typename Half<T>::type M;
  constexpr int BN = 32 * TN * WN, BM = 32 * TM * WM, PARTS = kParts<T>;
  static_assert(BM == kTileM && WM * WN * kWave == kGemmThreads);
  // A stage of LDS: STEP k of all parts of both tiles.  fp32's three parts are there together, so that each meets the others from LDS (six products of
  // what is loaded once; pairs of parts one after another load everything twice, and 257 rows' d_hidden came at the last-level cache's 6.5 TB/s).
  constexpr int STEP = kStep<T>, ROW = STEP * 2, PIECES = ROW / 16, PART = (BM + BN) * ROW, STAGE = PARTS * PART;
  // As many stages as fit, all but one of them on their way while that one is used.
  constexpr int STAGES = 155648 / STAGE < 4 ? 155648 / STAGE : 4;
  constexpr int LOAD_ROWS = 1024 / ROW;  // rows of a wave's load
  constexpr int LOADS_X = BM / LOAD_ROWS / 8, Y_WAVES = BN / LOAD_ROWS < 8 ? BN / LOAD_ROWS : 8, LOADS_Y = BN / LOAD_ROWS / Y_WAVES;  // per wave and part
  __shared__ __align__(16) unsigned char lds[STAGES * STAGE];

  const int lane = threadIdx.x % kWave, wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
  const int wm = wave / WN, wn = wave % WN;
  // Tiles with rows that count, a run of them to each XCD (blocks go to XCDs in turn), four n by m after m: what an XCD's blocks read together lies in
  // its L2 as often as can be.  (The last 64 rows' d is made past the count too, as zeros: the second products sum over whole steps.)
  const int32_t count = *q.count;
  const int n_there = JOB == kWeightGrad ? q.n_tiles : static_cast<int>(ceil_div(JOB == kDiffs ? ceil_div(count, kTileK) * kTileK : count, BN));
  const int tiles = q.m_tiles * n_there, xcd = blockIdx.x % q.xcds, local = blockIdx.x / q.xcds;
  int steps = q.steps;
  if (JOB == kWeightGrad) steps = static_cast<int>(ceil_div(count, kTileK)) * (kTileK / STEP);
  int tile, last_tile, slot = 0, from = 0, to = steps;  // a block that helps goes through more tiles than one
  Shares shares{tiles, 0, 1, 0};
  if constexpr (JOB == kRowGrad) shares = shares_of(tiles, q.cus, q.all_steps);
  const int each = static_cast<int>(ceil_div(shares.whole, q.xcds));
  if (local < each) {
    tile = xcd * each + local;
    if (tile >= shares.whole) return;
    last_tile = tile;
  } else {
    const int rest = shares.rest, items = shares.per == 0 ? rest * shares.slots : rest + static_cast<int>(ceil_div(rest, shares.per));
    const int each_rest = static_cast<int>(ceil_div(items, q.xcds)), item = xcd * each_rest + local - each;
    if (JOB != kRowGrad || local - each >= each_rest || item >= items) return;
    if (shares.per == 0) {
      slot = item / rest, tile = last_tile = shares.whole + item - slot * rest;
      const int span = static_cast<int>(ceil_div(steps, shares.slots));
      from = min(slot * span, steps), to = min(from + span, steps);
    } else {
      const int split = steps * shares.per / (shares.per + 1);
      if (item < rest) tile = last_tile = shares.whole + item, to = split;
      else slot = 1, tile = shares.whole + (item - rest) * shares.per, last_tile = min(tile + shares.per, tiles) - 1, from = split;
    }
  }
#pragma unroll 1
  for (;; ++tile) {
    const int first_n = tile / (4 * q.m_tiles) * 4, wide = min(4, n_there - first_n), inside = tile - first_n * q.m_tiles;
    const int mt = inside / wide, nt = first_n + inside % wide;
    const int m0 = mt * BM, n0 = nt * BN;

    // Addresses: a wave's load covers LOAD_ROWS rows; lane l brings the piece that belongs at its place.
    uint32_t off_x[LOADS_X], off_y[LOADS_Y];
    const auto turn = [](int row) { return PIECES == 8 ? row / 2 % 8 : row / 4 % 4; };
    const auto offset = [&](int row, int tile0, const Operand& o) {
      return static_cast<uint32_t>(min(tile0 + row, o.rows - 1) - tile0) * static_cast<uint32_t>(o.ld * 2) + static_cast<uint32_t>((lane % PIECES ^ turn(row)) * 16);
    };
#pragma unroll
    for (int i = 0; i < LOADS_X; ++i) off_x[i] = offset((wave * LOADS_X + i) * LOAD_ROWS + lane / PIECES, m0, q.x);
#pragma unroll
    for (int i = 0; i < LOADS_Y; ++i) off_y[i] = offset((wave * LOADS_Y + i) * LOAD_ROWS + lane / PIECES, n0, q.y);
    const char* const base_x = static_cast<const char*>(q.x.at) + static_cast<int64_t>(m0) * q.x.ld * 2;
    const char* const base_y = static_cast<const char*>(q.y.at) + static_cast<int64_t>(n0) * q.y.ld * 2;
    const int total = to - from;
    auto load_stage = [&](int s) {
      const int64_t k_bytes = static_cast<int64_t>(from + s) * ROW;
      unsigned char* to_lds = lds + s % STAGES * STAGE;
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        const auto rx = buffer_at(base_x + part * q.x.part * 2 + k_bytes), ry = buffer_at(base_y + part * q.y.part * 2 + k_bytes);
#pragma unroll
        for (int i = 0; i < LOADS_X; ++i) load_to_lds(rx, off_x[i], to_lds + part * PART + (wave * LOADS_X + i) * 1024);
        if (Y_WAVES == 8 || wave < Y_WAVES)
#pragma unroll
          for (int i = 0; i < LOADS_Y; ++i) load_to_lds(ry, off_y[i], to_lds + part * PART + BM * ROW + (wave * LOADS_Y + i) * 1024);
      }
    };

    f32x16 acc[TM][TN];
#pragma unroll
    for (int i = 0; i < TM; ++i)
#pragma unroll
      for (int j = 0; j < TN; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) acc[i][j][r] = 0.0f;

    const int r32 = lane % 32, half = lane / 32;
#pragma unroll
    for (int s = 0; s < STAGES - 1; ++s)
      if (s < total) load_stage(s);
    for (int s = 0; s < total; ++s) {
      if (STAGES == 2 || s + STAGES - 2 >= total) wait_loads<0>();
      else if (Y_WAVES == 8 || wave < Y_WAVES) wait_loads<(STAGES - 2) * PARTS * (LOADS_X + LOADS_Y)>();
      else wait_loads<(STAGES - 2) * PARTS * LOADS_X>();
      __builtin_amdgcn_s_barrier();
      asm volatile("" ::: "memory");
      if (s + STAGES - 1 < total) load_stage(s + STAGES - 1);
      const unsigned char* at = lds + s % STAGES * STAGE;
#pragma unroll
      for (int kk = 0; kk < STEP / 16; ++kk) {
        u32x4 x[PARTS][TM], y[PARTS][TN];
        const int piece = 2 * kk + half;
#pragma unroll
        for (int part = 0; part < PARTS; ++part) {
#pragma unroll
          for (int i = 0; i < TM; ++i) {
            const int row = (wm * TM + i) * 32 + r32;
            x[part][i] = *reinterpret_cast<const u32x4*>(at + part * PART + row * ROW + (piece ^ turn(row)) * 16);
          }
#pragma unroll
          for (int j = 0; j < TN; ++j) {
            const int row = (wn * TN + j) * 32 + r32;
            y[part][j] = *reinterpret_cast<const u32x4*>(at + part * PART + BM * ROW + row * ROW + (piece ^ turn(row)) * 16);
          }
        }
        // (the smallest products first: x3 y1, x2 y2, x1 y3, x2 y1, x1 y2, x1 y1)
#pragma unroll
        for (int sum = PARTS - 1; sum >= 0; --sum)
#pragma unroll
          for (int px = sum; px >= 0; --px)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int j = 0; j < TN; ++j) acc[i][j] = mma<M>(x[px][i], y[sum - px][j], acc[i][j]);
      }
    }

    // Element r of acc[i][j]: m = m0 + 32 (wm TM + i) + 8 (r / 4) + 4 half + r % 4,  n = n0 + 32 (wn TN + j) + r32.
    auto m_of = [&](int i, int r) { return 32 * (wm * TM + i) + 8 * (r / 4) + 4 * half + r % 4; };
    if constexpr (JOB == kSums) {
      __syncthreads();
      float* join_at = reinterpret_cast<float*>(lds);  // [WM][3][BN]
      const int64_t left = q.vocab - q.column0 - m0;   // columns of the tile that are there
      if (PARTS > 1 && q.kept != nullptr)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          const int n = n0 + 32 * (wn * TN + j) + r32;
          if (n < count)
#pragma unroll
            for (int i = 0; i < TM; ++i)
#pragma unroll
              for (int r4 = 0; r4 < 4; ++r4) {
                typedef float Four __attribute__((ext_vector_type(4)));
                *reinterpret_cast<Four*>(q.kept + static_cast<int64_t>(n) * q.ld_kept + m0 + m_of(i, 4 * r4)) =
                    Four{acc[i][j][4 * r4], acc[i][j][4 * r4 + 1], acc[i][j][4 * r4 + 2], acc[i][j][4 * r4 + 3]};
              }
        }
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + 32 * (wn * TN + j) + r32;
        const int64_t tok = n < count ? q.token[n] - q.column0 - m0 : -1;
        float m = -INFINITY;
        if (left < BM)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (m_of(i, r) >= left) acc[i][j][r] = -INFINITY;
        if (__any(tok >= 0 && tok < BM))
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (m_of(i, r) == tok) q.x_token[n] = acc[i][j][r];
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) m = fmaxf(m, acc[i][j][r]);
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
        const float m = live ? q.row_m[n] : 0.0f, inv = live ? q.row_inv_s[n] * kLift<T> : 0.0f;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) {
            const float p = __builtin_amdgcn_exp2f((acc[i][j][r] - m) * q.c) * inv;
            acc[i][j][r] = live && m_of(i, r) < left ? p : 0.0f;
          }
        if (__any(tok >= 0 && tok < BM))
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r)
              if (m_of(i, r) == tok) acc[i][j][r] -= kLift<T>;
      }
      // Both layouts leave through LDS in 16-byte pieces: rows n of the tile's m, piece p at place p ^ n % 16 of its row.  (Rows of a tile past the gathered
      // ones leave too, as zeros; columns up to the tile's end as well.)
      static_assert(BN * BM * 2 <= STAGES * STAGE);
      M* const rows = reinterpret_cast<M*>(lds);
      const auto at = [](int n, int piece) { return n * BM + (piece ^ n % 16) * 8; };
#pragma unroll
      for (int part = 0; part < PARTS; ++part) {
        __syncthreads();
#pragma unroll
        for (int j = 0; j < TN; ++j)
#pragma unroll
          for (int i = 0; i < TM; ++i)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
              typedef M Four __attribute__((ext_vector_type(4)));
              Four f;
#pragma unroll
              for (int r = 0; r < 4; ++r) {
                f[r] = static_cast<M>(acc[i][j][4 * r4 + r]);
                if (part + 1 < PARTS) acc[i][j][4 * r4 + r] -= static_cast<float>(f[r]);
              }
              *reinterpret_cast<Four*>(rows + at(32 * (wn * TN + j) + r32, 4 * (wm * TM + i) + r4) + 4 * half) = f;
            }
        __syncthreads();
        if (q.d != nullptr) {
          M* const to = static_cast<M*>(q.d) + part * q.d_part + m0;
          for (int k = threadIdx.x; k < BN * (BM / 8); k += kGemmThreads) {
            const int n = k / (BM / 8), piece = k % (BM / 8);
            if (n0 + n < q.n) *reinterpret_cast<u32x4*>(to + static_cast<int64_t>(n0 + n) * q.ld_d + piece * 8) = *reinterpret_cast<const u32x4*>(rows + at(n, piece));
          }
        }
        if (q.d_turned != nullptr) {
          M* const to = static_cast<M*>(q.d_turned) + part * q.t_part + n0;
          for (int k = threadIdx.x; k < (BN / 8) * (BM / 8); k += kGemmThreads) {
            const int n = k % (BN / 8) * 8, piece = k / (BN / 8);
            if (n0 + n >= q.n) continue;  // (q.n is a multiple of 64)
            u32x4 x[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = *reinterpret_cast<const u32x4*>(rows + at(n + e, piece));
#pragma unroll
            for (int e = 0; e < 8; ++e) {
              u32x4 y;
#pragma unroll
              for (int w = 0; w < 4; ++w) y[w] = __builtin_amdgcn_perm(x[2 * w + 1][e / 2], x[2 * w][e / 2], e % 2 != 0 ? 0x07060302u : 0x05040100u);
              *reinterpret_cast<u32x4*>(to + static_cast<int64_t>(m0 + piece * 8 + e) * q.ld_t + n) = y;
            }
          }
        }
      }
    } else if constexpr (JOB == kRowGrad) {
      static_assert(TM == WN && TN == (BN == 32 ? 1 : 2));  // as sum_at()
      // The sums lie as the lanes hold them, so that they are read and written whole (in rows, 16 bytes a row each time, a piece of 605 us for 16,384 columns
      // of 6,144 rows of 2,048 took 140 of them for that): see sum_at().
      typedef float Four __attribute__((ext_vector_type(4)));
      const int area = slot == 0 ? tile : tiles + (tile - shares.whole) * (shares.slots - 1) + slot - 1;
      Four* at = reinterpret_cast<Four*>(q.partial + static_cast<int64_t>(area) * (BN * BM)) + threadIdx.x;
#pragma unroll
      for (int i = 0; i < TM; ++i)
#pragma unroll
        for (int j = 0; j < TN; ++j) {
          Four before[4];
          if (q.add != 0)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) before[r4] = at[r4 * kGemmThreads];
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            Four sum;
#pragma unroll
            for (int r = 0; r < 4; ++r) sum[r] = acc[i][j][4 * r4 + r] * (1.0f / kLift<T>);
            at[r4 * kGemmThreads] = q.add != 0 ? before[r4] + sum : sum;
          }
          at += 4 * kGemmThreads;
        }
    } else {
      const float factor = 1.0f / kLift<T> * (q.inv_temp / (q.denom > 0.0f ? q.denom : static_cast<float>(max(count, 1))));
#pragma unroll
      for (int j = 0; j < TN; ++j) {
        const int n = n0 + 32 * (wn * TN + j) + r32;
        if (n >= q.n) continue;
#pragma unroll
        for (int i = 0; i < TM; ++i)
#pragma unroll
          for (int r4 = 0; r4 < 4; ++r4) {
            const int m = m0 + m_of(i, 4 * r4);
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
    if (JOB != kRowGrad || tile == last_tile) break;
    __syncthreads();  // the next tile's stages come where this one's are read
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
  int32_t cus, all_steps, n_tile;  // as d_hidden's products
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
    if (r < q.a.rows && tok < 0) {
      if (q.a.logp != nullptr) q.a.logp[r] = 0.0f;
      if (q.a.entropy != nullptr) q.a.entropy[r] = 0.0f;
    }
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
  void* turned;              // [part][dim][ld_turned]
  int64_t ld_turned, turned_part;
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
// A block: some thousand elements of whole rows (80,542 rows of 64, a row a block: 22 us for 21 MB, so 10).
int64_t pack_rows(int64_t ld_dst) { return std::max<int64_t>(1, 4 * kPackThreads / ld_dst); }
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_pack_kernel(const PackArgs q, int rows_each) {
  typedef typename Half<T>::type M;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * rows_each;
  const int64_t rows = q.count != nullptr ? static_cast<int64_t>(*q.count) : q.rows;
  const uint32_t width = static_cast<uint32_t>(q.ld_dst), all = static_cast<uint32_t>(min(static_cast<int64_t>(rows_each), q.out_rows - row0)) * width;
#pragma unroll 4
  for (uint32_t i = threadIdx.x; i < all; i += kPackThreads) {
    const int64_t row = row0 + i / width;
    const uint32_t k = i % width;
    float x = 0.0f;
    if (row < rows && k < q.dim) x = static_cast<float>(static_cast<const T*>(q.src)[(q.source != nullptr ? q.source[row] : row) * q.ld + k]);
    store_parts<T>(static_cast<M*>(q.dst) + row * q.ld_dst + k, q.part, x);
  }
}

// turned[k][row], and dst[row][k] where it is wanted: 64 x 64 tiles through LDS.
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_turn_kernel(const PackArgs q) {
  typedef typename Half<T>::type M;
  const int64_t rows = q.count != nullptr ? static_cast<int64_t>(*q.count) : q.rows;
  const int64_t row0 = static_cast<int64_t>(blockIdx.x) * 64, k0 = static_cast<int64_t>(blockIdx.y) * 64;
  if constexpr (sizeof(T) == 2) {
    // 16 bytes a lane on either side; in LDS rows of 66 elements, whose columns lie on as many banks
    __shared__ T half_tile[64][66];
    const int piece = threadIdx.x % 8 * 8, first = threadIdx.x / 8;
    const bool whole = k0 + 64 <= q.dim;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t row = row0 + first + 32 * i;
      RawPiece x{};
      if (row < rows) {
        const T* from = static_cast<const T*>(q.src) + (q.source != nullptr ? q.source[row] : row) * q.ld + k0 + piece;
        if (whole) x = load_raw(from);
        else
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (k0 + piece + e < q.dim) x.w[e / 2] |= static_cast<uint32_t>(__builtin_bit_cast(uint16_t, from[e])) << (e % 2 * 16);
      }
#pragma unroll
      for (int e = 0; e < 4; ++e) *reinterpret_cast<uint32_t*>(&half_tile[first + 32 * i][piece + 2 * e]) = x.w[e];
      if (q.dst != nullptr && row < q.out_rows) *reinterpret_cast<RawPiece*>(static_cast<T*>(q.dst) + row * q.ld_dst + k0 + piece) = x;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int64_t k = k0 + first + 32 * i;
      if (k >= q.dim) continue;
      RawPiece x;
#pragma unroll
      for (int e = 0; e < 4; ++e)
        x.w[e] = static_cast<uint32_t>(__builtin_bit_cast(uint16_t, half_tile[piece + 2 * e][first + 32 * i])) |
                 static_cast<uint32_t>(__builtin_bit_cast(uint16_t, half_tile[piece + 2 * e + 1][first + 32 * i])) << 16;
      *reinterpret_cast<RawPiece*>(static_cast<T*>(q.turned) + k * q.ld_turned + row0 + piece) = x;
    }
    return;
  }
  __shared__ float tile[64][65];
  const int lane = threadIdx.x % 64, part = threadIdx.x / 64;
  float x[16];
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t row = row0 + part + 4 * i, k = k0 + lane;
    x[i] = 0.0f;
    if (row < rows && k < q.dim) x[i] = static_cast<float>((static_cast<const T*>(q.src) + (q.source != nullptr ? q.source[row] : row) * q.ld)[k]);
  }
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    tile[part + 4 * i][lane] = x[i];
    if (q.dst != nullptr && row0 + part + 4 * i < q.out_rows) store_parts<T>(static_cast<M*>(q.dst) + (row0 + part + 4 * i) * q.ld_dst + k0 + lane, q.part, x[i]);
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int64_t k = k0 + part + 4 * i;
    if (k < q.dim) store_parts<T>(static_cast<M*>(q.turned) + k * q.ld_turned + row0 + lane, q.turned_part, tile[lane][part + 4 * i]);
  }
}

// d from products that were kept: 64 x 64 tiles, in both layouts.
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_diffs_kernel(const GemmArgs q) {
  typedef typename Half<T>::type M;
  __shared__ float tile[64][65];
  const int32_t count = *q.count;
  const int m0 = blockIdx.x * 64, n0 = blockIdx.y * 64;
  if (n0 >= count) return;
  const int lane = threadIdx.x % 64, part = threadIdx.x / 64;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    const int n = n0 + part + 4 * i, m = m0 + lane;
    float v = 0.0f;
    if (n < count && m < q.vocab) {
      const float p = __builtin_amdgcn_exp2f((q.kept[static_cast<int64_t>(n) * q.ld_kept + m] - q.row_m[n]) * q.c) * q.row_inv_s[n];
      v = (p - (m == q.token[n] ? 1.0f : 0.0f)) * kLift<T>;
    }
    tile[part + 4 * i][lane] = v;
    if (q.d != nullptr) store_parts<T>(static_cast<M*>(q.d) + static_cast<int64_t>(n) * q.ld_d + m, q.d_part, v);
  }
  if (q.d_turned == nullptr) return;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 16; ++i)
    store_parts<T>(static_cast<M*>(q.d_turned) + static_cast<int64_t>(m0 + part + 4 * i) * q.ld_t + n0 + lane, q.t_part, tile[lane][part + 4 * i]);
}

// ---- rows: the tiles' sums joined, log-probabilities, the loss ----

// The sums st and et relative to mt, added to those relative to m >= mt.  (Without columns, st = 0, they are nothing.)
__device__ __forceinline__ void add_sums(float& s, float& e, float m, float mt, float st, float et, float c) {
  if (st == 0.0f) return;
  const float d = mt == m ? 0.0f : fmaxf((mt - m) * c, kFloor), f = __builtin_amdgcn_exp2f(d);
  s = fmaf(st, f, s);
  e = fmaf(et + st * d, f, e);
}

// A block: 16 rows (the tiles' sums of a row lie rows apart, so neighbouring lanes take neighbouring rows) by 64 groups of tiles, so that 512 tiles (131,072
// columns) are one round of loads (16 groups, four rounds: 8 rows 11.6 us, so 8).
constexpr int kJoinThreads = 1024, kJoinRows = 16, kJoinGroups = kJoinThreads / kJoinRows;
__global__ __launch_bounds__(kJoinThreads) void linear_join_kernel(const RowArgs q) {
  __shared__ float part_m[kJoinGroups][kJoinRows], part_s[kJoinGroups][kJoinRows], part_e[kJoinGroups][kJoinRows];
  const int32_t count = *q.count;
  const int row = threadIdx.x % kJoinRows, group = threadIdx.x / kJoinRows;
  const int64_t n = static_cast<int64_t>(blockIdx.x) * kJoinRows + row;
  if (n - row >= count) return;
  const int64_t from = min(n, static_cast<int64_t>(count) - 1);
  constexpr int AHEAD = 8;  // tiles in flight
  float m = -INFINITY, s = 0.0f, e = 0.0f;
  for (int64_t t = group; t < q.tiles; t += kJoinGroups * AHEAD) {
    float mt[AHEAD], st[AHEAD], et[AHEAD];
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) {
      const int64_t at = min(t + u * kJoinGroups, q.tiles - 1) * q.sum_rows + from;
      mt[u] = q.tile_m[at], st[u] = q.tile_s[at], et[u] = q.tile_e[at];
    }
    const float before = m;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) m = fmaxf(m, mt[u]);
    const float d = before == m ? 0.0f : fmaxf((before - m) * q.c, kFloor), f = __builtin_amdgcn_exp2f(d);
    e = (e + s * d) * f;
    s *= f;
#pragma unroll
    for (int u = 0; u < AHEAD; ++u) add_sums(s, e, m, mt[u], t + u * kJoinGroups < q.tiles ? st[u] : 0.0f, et[u], q.c);
  }
  part_m[group][row] = m, part_s[group][row] = s, part_e[group][row] = e;
  for (int half = kJoinGroups / 2; half > 0; half /= 2) {  // (in pairs: the same order every time)
    __syncthreads();
    if (group >= half) continue;
    const float mo = part_m[group + half][row], before = m;
    m = fmaxf(m, mo);
    float s2 = 0.0f, e2 = 0.0f;
    add_sums(s2, e2, m, before, s, e, q.c);
    add_sums(s2, e2, m, mo, part_s[group + half][row], part_e[group + half][row], q.c);
    s = s2, e = e2;
    part_m[group][row] = m, part_s[group][row] = s, part_e[group][row] = e;
  }
  if (group != 0 || n >= count) return;
  const float log2_s = log2f(s), lp = kLn2 * ((q.x_token[n] - m) * q.c - log2_s), h = kLn2 * (log2_s - e / s);
  q.row_m[n] = m, q.row_inv_s[n] = 1.0f / s, q.row_lp[n] = lp, q.row_h[n] = h;
  const int32_t r = q.source[n];
  if (q.a.logp != nullptr) q.a.logp[r] = lp;
  if (q.a.entropy != nullptr) q.a.entropy[r] = h;
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

// Where linear_gemm_kernel's lanes leave a tile's sums of n and of m .. m + 3, m a multiple of 4.
__device__ __forceinline__ int sum_at(int n, int m, int n_tile) {
  const int tn = n_tile == 32 ? 1 : 2, wn = n_tile / (32 * tn), tm = wn;  // (256 m by 8 / wn waves of tm tiles of 32)
  const int thread = (m / (32 * tm) * wn + n / (32 * tn)) * kWave + m / 4 % 2 * 32 + n % 32;
  return (((m / 32 % tm * tn + n / 32 % tn) * 4 + m / 8 % 4) * kGemmThreads + thread) * 4;
}

// d_hidden: the shares' sums of each row, zeros where a row does not count.  A block takes 8 rows, whose sums lie side by side if they all count (a row a block
// reads eighths of lines: 107 us for 6,144 rows of 2,048).
constexpr int kGradRows = 8, kGradColumns = kPackThreads / kGradRows * 4;
template <class T>
__global__ __launch_bounds__(kPackThreads) void linear_row_grad_kernel(const RowArgs q) {
  typedef float Four __attribute__((ext_vector_type(4)));
  const int64_t r = static_cast<int64_t>(blockIdx.x) * kGradRows + threadIdx.x % kGradRows;
  if (r >= q.a.rows) return;
  const int32_t n = q.gathered[r];
  T* to = static_cast<T*>(q.a.d_hidden) + r * q.a.ld_d_hidden;
  const float factor = static_cast<float>(1.0 / (q.a.temperature * (q.a.denom > 0.0 ? q.a.denom : static_cast<double>(max(*q.count, 1)))));
  const int n_there = static_cast<int>(ceil_div(*q.count, q.n_tile)), m_tiles = static_cast<int>(ceil_div(q.a.dim, kTileM)), tiles = m_tiles * n_there;
  const Shares shares = shares_of(tiles, q.cus, q.all_steps);
  const int nt = n / q.n_tile, first_n = nt / 4 * 4, wide = min(4, n_there - first_n);
  const int64_t area = static_cast<int64_t>(q.n_tile) * kTileM;
#pragma unroll 4
  for (int k = blockIdx.y * kGradColumns + threadIdx.x / kGradRows * 4; k < q.a.dim; k += gridDim.y * kGradColumns) {
    Four x{};
    if (n >= 0) {
      const int tile = first_n * m_tiles + k / kTileM * wide + nt - first_n, slots = tile < shares.whole ? 0 : shares.slots - 1;
      const float* at = q.partial + tile * area + sum_at(n % q.n_tile, k % kTileM, q.n_tile);
      x = *reinterpret_cast<const Four*>(at);
      at += (tiles - tile + static_cast<int64_t>(tile - shares.whole) * slots) * area;
      constexpr int AHEAD = 8;
      for (int s = 0; s < slots; s += AHEAD) {
        Four y[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) y[u] = *reinterpret_cast<const Four*>(at + min(s + u, slots - 1) * area);
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
          if (s + u < slots) x += y[u];
      }
    }
    if (k + 4 <= q.a.dim) {
      typedef T Out __attribute__((ext_vector_type(4), aligned(sizeof(T))));
      Out o;
#pragma unroll
      for (int e = 0; e < 4; ++e) o[e] = static_cast<T>(x[e] * factor);
      *reinterpret_cast<Out*>(to + k) = o;
    } else {
#pragma unroll
      for (int e = 0; e < 4; ++e)
        if (k + e < q.a.dim) to[k + e] = static_cast<T>(x[e] * factor);
    }
  }
}

// ---- the host's part ----

struct Plan {
  int64_t rows, k, piece, pieces;  // rows and k padded to whole tiles of k
  int parts, cus, n_tile;
  bool direct;  // the weight is an operand as it lies
  bool keep;    // the products of the one piece are kept
  size_t count, source, gathered, token, sums, x_token, row, hidden, hidden_turned, weight, weight_turned, d, d_turned, partial, kept, bytes;
};

int64_t up(int64_t x, int64_t to) { return ceil_div(x, to) * to; }

// Narrower tiles of n where their blocks, too, find a compute unit each (4,524 rows, 6,290 columns of 33: the weight's gradient in 25 blocks of 256 columns
// 95 us, in 197 of 32 36).
int narrow(int n_tile, int64_t m_tiles, int64_t n, int64_t cus) {
  if (n_tile == 256 && 2 * m_tiles * ceil_div(n, 256) <= cus) n_tile = 128;
  if (n_tile == 128 && 4 * m_tiles * ceil_div(n, 128) <= cus) n_tile = 32;
  return n_tile;
}

Plan plan_of(const ppo_linear_loss_args& a, bool gradient) {
  Plan p{};
  int64_t cus = device_info().cus;
  if (cus <= 0) cus = 256;
  p.parts = a.type == PPO_TYPE_F32 ? kMaxParts : 1;
  p.rows = up(std::max<int64_t>(a.rows, 1), kTileK);
  p.k = up(a.dim, kTileK);
  p.direct = a.type != PPO_TYPE_F32 && a.dim % kTileK == 0 && a.ld_weight % 8 == 0 && reinterpret_cast<uintptr_t>(a.weight) % 16 == 0;
  const int64_t column = 2 * p.parts * ((gradient ? (a.d_hidden != nullptr) + (a.d_weight != nullptr) : 0) * p.rows + (p.direct ? 0 : p.k) +
                                         (gradient && a.d_hidden != nullptr ? a.dim : 0));
  // rows of a tile: few rows' tiles hold nothing else, three fp32 parts of 256 do not fit into LDS (131,072 columns of 1,024, bf16: 32 rows 56 us in tiles of 32, 60
  // of 128; 128 rows 63 of 128, 82 of 256; 200 rows 92 and 84; 384 rows 130 and 143; 512 rows 167 and 145)
  p.n_tile = a.rows <= 32 ? 32 : a.type == PPO_TYPE_F32 || a.rows <= 128 || (a.rows > 256 && a.rows <= 384) ? 128 : 256;
  p.n_tile = narrow(p.n_tile, ceil_div(a.vocab, kTileM), a.rows, cus);
  int64_t piece = kPieceBytes / std::max<int64_t>(column, 1) / kTileM * kTileM;
  piece = std::min(std::max(piece, kMinPiece), int64_t{1} << 21);  // (a tile of d's offsets stay in 31 bits)
  if (!gradient && p.direct) piece = up(a.vocab, kTileM);
  piece = std::min(piece, kMostTiles / ceil_div(p.rows, p.n_tile) * kTileM);
  if (gradient) piece = std::min(piece, kMostTiles / (2 * ceil_div(a.dim, kTileM)) * kTileM);
  p.piece = std::min(piece, up(a.vocab, kTileM));
  p.pieces = ceil_div(a.vocab, p.piece);
  if (p.pieces > 1) {
    // columns whose d_weight takes whole rounds of the chip's blocks, or else pieces of one size (8,192 x 131,072 of 2,048: 16,384 columns 512 blocks and two rounds,
    // 18,944 592 blocks and three)
    const int64_t blocks = ceil_div(a.dim, kTileM), round = cus / std::gcd(cus, blocks) * kTileM;
    p.piece = p.piece >= round ? p.piece / round * round : up(ceil_div(a.vocab, p.pieces), kTileM);
    p.pieces = ceil_div(a.vocab, p.piece);
  }
  p.cus = static_cast<int>(cus);
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
  // fp32 products come six times as dear as 16-bit ones: where one piece holds the vocabulary and its products are small, they are kept for d instead of
  // made again (257 rows of 515 over 50,021 columns: 121 us again, 34 from what was kept; bf16 products are made in the time that reading takes)
  p.keep = gradient && a.type == PPO_TYPE_F32 && p.pieces == 1 && p.rows * p.piece * 4 <= kKeptBytes && (a.d_hidden != nullptr || a.d_weight != nullptr);
  p.kept = room(p.keep ? p.rows * p.piece * 4 : 0);
  if (gradient) {
    if (a.d_hidden != nullptr) {
      p.weight_turned = room(p.parts * a.dim * p.piece * 2);
      p.d = room(p.parts * p.rows * p.piece * 2);
      p.partial = room((ceil_div(p.rows, p.n_tile) * ceil_div(a.dim, kTileM) + cus) * p.n_tile * kTileM * 4);  // (shares_of(): more than one less than cus times)
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
  g.m_tiles = static_cast<int32_t>(ceil_div(g.m, kTileM));
  if (JOB == kWeightGrad) n_tile = narrow(sizeof(T) == 4 ? 128 : 256, g.m_tiles, g.n, g.cus);  // n is the vocabulary there
  g.n_tiles = static_cast<int32_t>(ceil_div(g.n, n_tile));
  g.xcds = std::max(1, device_info().xcds);
  const dim3 grid(static_cast<uint32_t>(up(static_cast<int64_t>(g.m_tiles) * g.n_tiles, g.xcds) + (JOB == kRowGrad ? up(g.cus, g.xcds) : 0)));
#define PPO_GEMM(...) hipLaunchKernelGGL((linear_gemm_kernel<T, __VA_ARGS__, JOB>), grid, dim3(kGemmThreads), 0, st, g)
  if constexpr (sizeof(T) == 2)
    if (n_tile == 256) PPO_GEMM(2, 4, 4, 2);
  if (n_tile == 128) PPO_GEMM(4, 2, 2, 2);
  if (n_tile == 32) PPO_GEMM(8, 1, 1, 1);
#undef PPO_GEMM
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
  r.cus = p.cus, r.all_steps = static_cast<int32_t>(p.piece / kStep<T>), r.n_tile = p.n_tile;
  hipLaunchKernelGGL(linear_rows_kernel, dim3(1), dim3(kRowThreads), 0, st, r);
  if (int rc = check_launch("linear_rows_kernel")) return rc;

  const bool to_hidden = gradient && a.d_hidden != nullptr, to_weight = gradient && a.d_weight != nullptr;
  // Rows of `from` as an operand, turned, or both at once.
  auto pack = [&](const void* from, int64_t ld, int64_t n, bool gathered, void* to, int64_t part, void* turned, int64_t ld_turned, int64_t turned_part) -> int {
    const PackArgs w{from, ld, n, a.dim, gathered ? r.source : nullptr, gathered ? r.count : nullptr, to, p.k, part, n, turned, ld_turned, turned_part};
    if (turned != nullptr) {  // (up to p.k: the operand's padding is this launch's too)
      hipLaunchKernelGGL(linear_turn_kernel<T>, dim3(static_cast<uint32_t>(ceil_div(n, 64)), static_cast<uint32_t>(p.k / 64)), dim3(kPackThreads), 0, st, w);
      return check_launch("linear_turn_kernel");
    }
    hipLaunchKernelGGL(linear_pack_kernel<T>, dim3(static_cast<uint32_t>(ceil_div(n, pack_rows(p.k)))), dim3(kPackThreads), 0, st, w, static_cast<int>(pack_rows(p.k)));
    return check_launch("linear_pack_kernel");
  };
  if (int rc = pack(a.hidden, a.ld_hidden, p.rows, true, ws + p.hidden, p.rows * p.k, to_weight ? ws + p.hidden_turned : nullptr, p.rows, a.dim * p.rows)) return rc;

  GemmArgs g{};
  g.y = Operand{ws + p.hidden, p.k, p.rows * p.k, static_cast<int32_t>(p.rows)};
  g.n = static_cast<int32_t>(p.rows);
  g.steps = static_cast<int32_t>(p.k / kStep<T>);
  g.count = r.count;
  g.vocab = a.vocab;
  g.c = r.c;
  g.token = r.token;
  g.tile_m = r.tile_m, g.tile_s = r.tile_s, g.tile_e = r.tile_e, g.sum_rows = r.sum_rows;
  g.x_token = r.x_token;
  g.row_m = r.row_m, g.row_inv_s = r.row_inv_s;
  g.denom = static_cast<float>(a.denom);
  g.inv_temp = static_cast<float>(1.0 / a.temperature);
  g.kept = p.keep ? reinterpret_cast<float*>(ws + p.kept) : nullptr;
  g.ld_kept = p.piece;
  // A piece of the weight as an operand, and turned for d_hidden; `packed`: the operand is there.
  auto weight_piece = [&](int64_t v0, int64_t n, bool turn, bool packed) -> int {
    const char* from = static_cast<const char*>(a.weight) + v0 * a.ld_weight * size;
    g.m = static_cast<int32_t>(n);
    g.column0 = v0;
    if (p.direct) g.x = Operand{from, a.ld_weight, 0, static_cast<int32_t>(n)};
    else g.x = Operand{ws + p.weight, p.k, p.piece * p.k, static_cast<int32_t>(n)};
    void* to = p.direct || packed ? nullptr : ws + p.weight;
    if (to == nullptr && !turn) return PPO_OK;
    return pack(from, a.ld_weight, n, false, to, p.piece * p.k, turn ? ws + p.weight_turned : nullptr, p.piece, a.dim * p.piece);
  };
  const bool once = p.pieces == 1;  // then the copies that the sums need serve the gradients too
  for (int64_t v0 = 0; v0 < a.vocab && a.rows > 0; v0 += p.piece) {
    if (int rc = weight_piece(v0, std::min(p.piece, a.vocab - v0), once && to_hidden, false)) return rc;
    g.tile0 = v0 / kTileM;
    if (int rc = launch_gemm<T, kSums>(g, p.n_tile, st)) return rc;
  }
  if (a.rows > 0) {
    hipLaunchKernelGGL(linear_join_kernel, dim3(static_cast<uint32_t>(ceil_div(a.rows, kJoinRows))), dim3(kJoinThreads), 0, st, r);
    if (int rc = check_launch("linear_join_kernel")) return rc;
  }
  if (!gradient) return PPO_OK;
  hipLaunchKernelGGL(linear_stats_kernel, dim3(1), dim3(kRowThreads), 0, st, r);
  if (int rc = check_launch("linear_stats_kernel")) return rc;
  if (!to_hidden && !to_weight) return PPO_OK;

  for (int64_t v0 = 0; v0 < a.vocab; v0 += p.piece) {
    const int64_t n = std::min(p.piece, a.vocab - v0);
    if (a.rows > 0 && !once)
      if (int rc = weight_piece(v0, n, to_hidden, false)) return rc;
    const Operand hidden = g.y, weight = g.x;
    g.d = to_hidden ? ws + p.d : nullptr;
    g.d_turned = to_weight ? ws + p.d_turned : nullptr;
    g.ld_d = p.piece, g.d_part = p.rows * p.piece;
    g.ld_t = p.rows, g.t_part = p.piece * p.rows;
    if (a.rows > 0 && p.keep) {
      hipLaunchKernelGGL(linear_diffs_kernel<T>, dim3(static_cast<uint32_t>(up(n, kTileK) / 64), static_cast<uint32_t>(p.rows / 64)), dim3(kPackThreads), 0, st, g);
      if (int rc = check_launch("linear_diffs_kernel")) return rc;
    } else if (a.rows > 0) {
      if (int rc = launch_gemm<T, kDiffs>(g, p.n_tile, st)) return rc;
    }
    if (to_hidden && a.rows > 0) {
      GemmArgs b = g;
      b.x = Operand{ws + p.weight_turned, p.piece, a.dim * p.piece, static_cast<int32_t>(a.dim)};
      b.y = Operand{ws + p.d, p.piece, p.rows * p.piece, static_cast<int32_t>(p.rows)};
      b.m = static_cast<int32_t>(a.dim);
      b.steps = static_cast<int32_t>(up(n, kTileK) / kStep<T>);
      b.partial = reinterpret_cast<float*>(ws + p.partial);
      b.cus = p.cus, b.all_steps = r.all_steps;
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
      b.cus = p.cus;
      if (int rc = launch_gemm<T, kWeightGrad>(b, p.n_tile, st)) return rc;
    }
    g.x = weight, g.y = hidden;
  }
  if (to_hidden && a.rows > 0) {
    const int64_t blocks = ceil_div(a.rows, kGradRows), columns = std::min(ceil_div(a.dim, kGradColumns), ceil_div(4 * p.cus, blocks));
    hipLaunchKernelGGL(linear_row_grad_kernel<T>, dim3(static_cast<uint32_t>(blocks), static_cast<uint32_t>(columns)), dim3(kPackThreads), 0, st, r);
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
