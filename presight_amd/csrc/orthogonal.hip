// The orthogonalised update: a batch of matrices G [B, m, n], each scaled to Frobenius norm one and pushed `steps` times through the odd
// polynomial  X <- a X + (b S + c S^2) X,  S = X X^T,  that moves singular values towards one (Newton-Schulz).  X is kept short side
// first: [s, l] with s = min(m, n), l = max(m, n), so both products of a step with X and the square of S have the fewest operations.
//
// Arithmetic.  The polynomial multiplies what rounding leaves in the small singular directions by up to a^steps, so one 16-bit rounding
// per step is not enough for an fp32 result.  Every matrix is kept as a PAIR of fp16 planes, value = (hi + lo / 2048) / scale: 22 bits
// and the sign, and a product is three matrix instructions, hi hi + (hi lo + lo hi) / 2048, summed in fp32 (lo lo, 2^-24 of the product, is
// left out).  That is nearly fp32's precision at a third of the fp16 rate, three times the fp32 matrix rate (large products: 1463 and 154
// TFLOP/s).
//
// Range.  The planes hold X^ = X / r with r = norm / (norm + eps) at the start, so an input far below eps loses nothing; a step
// multiplies r by the power of two `grow` that bounds a + b t + c t^2, until r passes 1/2, and keeps it from then on.  The caller
// checks that the iterates' squared singular values and the polynomial stay under 15: with X^ <= 2 X the entries of X^ are below 7.75,
// those of S^ below 60 and those of the polynomial below 15, and each is scaled to the planes' end, 65504.  lo is 2048 times what hi leaves,
// so it is as far from the subnormal numbers as hi is: X^ has its 22 bits down to entries of 2^-27 (of the whole matrix' norm, at the start),
// and smaller ones are off by up to 2^-49.  (385 x 1290 normal numbers, one of them 10^6 times the rest: 5e-7 from 64 bits relative to the
// norm, plain fp32 3e-7; with lo in hi's units, subnormal below 2^-12, 8e-6.)
#include <type_traits>
#include "gemm_core.hpp"

namespace {

using namespace ps;

constexpr float kScaleX = 8192.0f, kScaleS = 1024.0f, kScaleP = 4096.0f;  // what the planes of X^, S^ and the polynomial hold of a value
constexpr float kLowScale = 2048.0f, kLowUnit = 1.0f / kLowScale;         // lo's part of hi's unit
constexpr int kCompute = 256;                                // compute units
constexpr int kNormParts = 256;                              // partial sums of squares per matrix, at most

template <typename V>  // float or double, scaled
__device__ __forceinline__ void split(V t, _Float16& hi, _Float16& lo) {
  hi = (_Float16)(float)t;
  lo = (_Float16)(float)((t - (V)(float)hi) * (V)kLowScale);
}

// The two planes lie side by side, 32 columns of hi and then the same 32 of lo: 128 bytes, a cache line and a tile row.  Rows are padded to
// whole lines of 64 columns.
__host__ __device__ inline int64_t pair_at(int col, int plane) { return (int64_t)(col >> 5) * 64 + plane * 32 + (col & 31); }

struct Shape {  // of one matrix
  int64_t m, n;      // as given
  int s, l;          // short and long side
  int sp, lp;        // rounded up to 64 (zeros there); rows of a pair are twice as long
  bool tall;         // m > n: X = G^T
};
Shape shape_of(int64_t m, int64_t n) {
  Shape h;
  h.m = m, h.n = n;
  h.tall = m > n;
  h.s = (int)(h.tall ? n : m);
  h.l = (int)(h.tall ? m : n);
  h.sp = (h.s + 63) & ~63;
  h.lp = (h.l + 63) & ~63;
  return h;
}

// Workspace of a batch
struct Work {
  _Float16 *x[2], *gram, *poly;  // pairs: [B][s][2 lp] twice, [B][s][2 sp], [B][s][2 sp]
  double* norms;                 // [B][parts]
  float* ratio;                  // [B] r at the start
  f32x4* shares;                 // [parts][B][tiles][64 x 64] fp32 sums, where a product's k is shared out
  int parts;
  int64_t bytes;
};
// Where the matrix comes from: G itself, or an optimizer's momentum buf <- mu buf + (1 - mu) g, taken as it is or (nesterov) as
// mu buf + (1 - mu) g once more
struct Source {
  const void* g;
  float* buf;  // null: g alone
  float mu, nu;  // momentum, 1 - momentum
  int nesterov;
};

template <bool MOMENTUM, bool UPDATE>
__device__ __forceinline__ float source_step(const Source& src, float g, float& b) {
#pragma clang fp contract(off)  // the same bits in both passes over the source
  if constexpr (!MOMENTUM) return g;
  if constexpr (UPDATE) b = src.mu * b + src.nu * g;
  return src.nesterov ? src.mu * b + src.nu * g : b;
}
template <typename T, bool MOMENTUM, bool UPDATE>
__device__ __forceinline__ float source_value(const Source& src, int64_t i) {
  float b = 0.0f;
  if constexpr (MOMENTUM) b = src.buf[i];
  const float v = source_step<MOMENTUM, UPDATE>(src, to_f32(reinterpret_cast<const T*>(src.g)[i]), b);
  if constexpr (MOMENTUM && UPDATE) src.buf[i] = b;
  return v;
}
// four consecutive values, zeros from the `left`th on
template <typename T, bool MOMENTUM, bool UPDATE>
__device__ __forceinline__ void source_pack(const Source& src, int64_t i, int64_t left, float (&v)[4]) {
  if (left < 4) {
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = k < left ? source_value<T, MOMENTUM, UPDATE>(src, i + k) : 0.0f;
    return;
  }
  const Pack<T, 4> g = load_any<T, 4>(reinterpret_cast<const T*>(src.g) + i);
  Pack<float, 4> b{};
  if constexpr (MOMENTUM) b = load_any<float, 4>(src.buf + i);
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = source_step<MOMENTUM, UPDATE>(src, to_f32(g.v[k]), b.v[k]);
  if constexpr (MOMENTUM && UPDATE) store_any(src.buf + i, b);
}

// 2048 x 4096 fp32: 13 us for 34 MB; with the momentum, 8 x 1024 x 2048: 35 us for 201 MB (5.7 TB/s, some of it from the last-level cache).
// partial sums of squares, in 64 bits: entries of any fp32 size neither overflow nor vanish
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_norm_kernel(Source src, int64_t size, Work w) {
  __shared__ double part[4];
  const int64_t base = (int64_t)blockIdx.y * size;
  double sum[4] = {};
  for (int64_t i = ((int64_t)blockIdx.x * 256 + threadIdx.x) * 4; i < size; i += (int64_t)gridDim.x * 256 * 4) {
    float v[4];
    source_pack<T, MOMENTUM, true>(src, base + i, size - i, v);
#pragma unroll
    for (int k = 0; k < 4; ++k) sum[k] += (double)v[k] * v[k];
  }
  double all = (sum[0] + sum[1]) + (sum[2] + sum[3]);
  for (int d = 32; d > 0; d >>= 1) all += __shfl_xor(all, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = all;
  __syncthreads();
  if (threadIdx.x == 0) w.norms[(int64_t)blockIdx.y * w.parts + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
}

// r before step i
__device__ __forceinline__ float ratio_at(float r, int i, float grow) {
  for (; i > 0; --i) {
    if (r * grow <= 1.0f) {
      r *= grow;
    } else {
      while (r > 0.0f && r * 2.0f <= 1.0f) r *= 2.0f;
    }
  }
  return r;
}

// 2048 x 4096 fp32: 25 us for 67 MB; 8 x 1024 x 2048 with the momentum: 48 us for 201 MB.
// X^ = G / norm as pairs [s][2 lp], 64 x 64 elements at a time (turned in LDS where G is tall); zeros in the padding
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_start_kernel(Source src, Shape h, Work w, float eps) {
  __shared__ _Float16 tile[2][64][72];  // (rows of 144 bytes: 16-byte chunks, 36 banks apart)
  __shared__ double inv_of;
  const int64_t b = blockIdx.z;
  if (threadIdx.x < 64) {
    double sum = 0.0;
    for (int i = threadIdx.x; i < w.parts; i += 64) sum += w.norms[b * w.parts + i];
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
    if (threadIdx.x == 0) {
      const double norm = sqrt(sum);
      inv_of = norm == 0.0 ? 0.0 : 1.0 / norm;
      if (blockIdx.x == 0 && blockIdx.y == 0) w.ratio[b] = norm == 0.0 ? 0.0f : (float)(norm / (norm + (double)eps));
    }
  }
  __syncthreads();
  const double inv = inv_of;
  const int r0 = blockIdx.y * 64, c0 = blockIdx.x * 64;  // of G
  const int64_t base = b * h.m * h.n;
#pragma unroll
  for (int id = threadIdx.x; id < 64 * 64 / 4; id += 256) {
    const int r = id / 16, c = id % 16 * 4;
    float v[4] = {};
    if (r0 + r < h.m && c0 + c < h.n) source_pack<T, MOMENTUM, false>(src, base + (int64_t)(r0 + r) * h.n + c0 + c, h.n - (c0 + c), v);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int row = h.tall ? c + k : r, col = h.tall ? r : c + k;
      split(v[k] * inv * (double)kScaleX, tile[0][row][col], tile[1][row][col]);
    }
  }
  __syncthreads();
  const int m0 = h.tall ? c0 : r0, n0 = h.tall ? r0 : c0;  // of X
  for (int id = threadIdx.x; id < 2 * 64 * 8; id += 256) {
    const int p = id >> 9, row = (id >> 3) & 63, col = (id & 7) * 8;
    if (m0 + row < h.s && n0 + col < h.lp)
      *reinterpret_cast<u32x4*>(w.x[0] + (b * h.s + m0 + row) * 2 * h.lp + pair_at(n0 + col, p)) = *reinterpret_cast<const u32x4*>(&tile[p][row][col]);
  }
}

// ------------------------------------------------------------------------------------------------ products of pairs
enum Product {
  kGram,   // S = X X^T                            rows of X     x rows of X,    k = l
  kPoly,   // P = a I + b S + c S S                rows of S     x rows of S,    k = s    (S is symmetric)
  kApply,  // X' = P X                             rows of P     x columns of X, k = s
  kLast    // ... of the last step: into the result
};

struct Result {  // of the last step
  void* out;      // [B, m, n] of the result's type, or the parameters [B, m, n] in fp32
  int update;     // parameters: p <- keep p - rate X
  float keep, rate;
};

struct Poly {
  double a, b, c;
  float grow;
};

struct Operands {  // pairs
  const _Float16 *a, *b;  // [B][ra][2 k]; [B][rb][2 k], or for kApply and kLast [B][k_rows][2 ldb]
  int ra, rb, k;          // k: padded, and half the rows' distance
  int k_rows, ldb;
};

// A workgroup's tile: BM x BN; a stage is 32 k of both planes of either operand, one tile row of 128 bytes for a row of k (KC).  A compute
// unit can have about 17 bytes per cycle of the L2's in flight, so the tile decides how fast the matrix instructions are fed: at their full
// rate 256 x 128 asks for 32 bytes per cycle, 128 x 128 for 43 and 64 x 64 for 85, and a step of k takes as long as its stage of 48, 32 or
// 16 KiB takes to arrive.  The two small products add up apart from the large one: each of their additions to it would cost it another rounding.
//
// 2048 x 4096: S 90 us, a I + b S + c S S 57, times X 99: 573, 452 and 1041 TFLOP/s of pairs' products (half of S and S S by symmetry, three
// products per pair), where a large fp16 product reaches 1463; 8 x 1024 x 2048: 87, 64 and 107 us.  A few tiles:
// 3 x 385 x 129 takes 7 to 9 us a product, most of it the launch, the first loads from memory that another XCD wrote, and the way out.
//
// The result leaves through LDS as rows of whole lines.  Of a symmetric one only what lies on and below the diagonal's BN x BN blocks is
// computed and written, and then written turned.
// Few tiles and a long k, as of S of a wide matrix: k is shared out over several workgroups per tile (kShare), their fp32 sums go through memory,
// and a second launch (kJoin) adds them up in order and takes the way out.  (All five steps: 512 x 8192 612 -> 301 us.)
enum Part { kAllOfK, kShare, kJoin };

constexpr int kPairK = 32;
template <int BM>
struct PairTile {
  static constexpr int kN = BM == 64 ? 64 : 128, kThreads = BM == 64 ? 256 : 512;
  static constexpr int kWaveM = BM == 64 ? 32 : 64, kWavesN = kThreads / 64 / (BM / kWaveM), kWaveN = kN / kWavesN;
  static constexpr int kStages = BM == 256 ? 3 : 4, kGroup = BM == 256 ? 1 : 2;  // in LDS; per barrier
  static constexpr int kStage = (BM + kN) * kTileRowBytes, kLds = kStages * kStage;
};

// a tile on its way out: rows of `bytes`, 16-byte chunks spread so that 16 rows at a time meet different banks
__device__ __forceinline__ int out_addr(int row, int bytes, int byte) { return row * bytes + (((byte >> 4) ^ (row & 15)) << 4) + (byte & 15); }

// tiles of a symmetric product in the row of tiles tm: those that reach the diagonal or below
__host__ __device__ inline int symmetric_tiles(int tm, int across, int n_tiles) {  // across: tiles' height over their width
  const int n = (tm + 1) * across;
  return n < n_tiles ? n : n_tiles;
}

template <typename T, Product WHAT, int BM, Part PART>
__global__ __launch_bounds__(PairTile<BM>::kThreads) void ns_product_kernel(Operands o, Shape h, Work w, int batches, int tiles, int parts, int step, Poly c,
                                                                            Result res) {
  using Tile = PairTile<BM>;
  constexpr int BN = Tile::kN, NT = Tile::kThreads, WN = Tile::kWavesN, MI = Tile::kWaveM / 16, NJ = Tile::kWaveN / 16, kStages = Tile::kStages,
                kStage = Tile::kStage, kGroup = Tile::kGroup;
  constexpr bool kSymmetric = WHAT == kGram || WHAT == kPoly;
  using SourceA = DirectSource<_Float16, BM, NT, false>;
  using SourceB = std::conditional_t<kSymmetric, DirectSource<_Float16, BN, NT, false>, DirectSource<_Float16, 2 * BN, NT, true, kPairK>>;
  constexpr int kLoads = decltype(SourceA::tile)::N + decltype(SourceB::tile)::N;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int m_tiles = (o.ra + BM - 1) / BM, n_tiles = (o.rb + BN - 1) / BN;
  // (the batch's matrices one under the other; `tiles`: of one of them)
  const int shares = PART == kShare ? parts : 1;
  int place = xcd_place(blockIdx.x, tiles * batches * shares), part = 0;
  if (place < 0) return;
  if constexpr (PART == kShare) {  // (a part's tiles share their operands)
    part = place / (tiles * batches);
    place -= part * tiles * batches;
  }
  int tm = 0, tn;
  int64_t batch;
  if constexpr (kSymmetric) {
    batch = place / tiles;
    tn = place % tiles;
    for (int n; tn >= (n = symmetric_tiles(tm, BM / BN, n_tiles)); ++tm) tn -= n;
  } else {
    const TileAt at = patched_tile(place, batches * m_tiles, n_tiles);
    batch = at.m / m_tiles;
    tm = at.m % m_tiles, tn = at.n;
  }
  const int m0 = tm * BM, n0 = tn * BN;
  const int rows = o.ra - m0 < BM ? o.ra - m0 : BM, cols = o.rb - n0 < BN ? o.rb - n0 : BN;
  // this part's steps, even numbers of them; the loads behind the last one bring zeros
  const int steps = o.k / kPairK, first = PART == kShare ? steps / 2 * part / parts * 2 : 0, end = PART == kShare ? steps / 2 * (part + 1) / parts * 2 : steps;
  const SourceA sa(o.a + (batch * o.ra + m0) * 2 * o.k, 2 * o.k, rows, 2 * kPairK * end);
  const SourceB sb = kSymmetric ? SourceB(o.b + (batch * o.rb + n0) * 2 * o.k, 2 * o.k, cols, 2 * kPairK * end)
                                : SourceB(o.b + batch * o.k_rows * 2 * o.ldb + 2 * n0, 2 * o.ldb, 2 * (o.ldb - n0), o.k_rows);
  auto load = [&](int stage) {  // stage by stage of k; KC counts both planes
    char* to = lds + stage % kStages * kStage;
    sa.load(stage * 2 * kPairK, to);
    sb.load(stage * (kSymmetric ? 2 : 1) * kPairK, to + BM * kTileRowBytes);
  };
  const int wave = threadIdx.x >> 6, wm = wave / WN * Tile::kWaveM, wn = wave % WN * Tile::kWaveN;
  f32x4 acc[MI][NJ], fine[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = fine[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  // what the result needs besides the sums is asked for before them (S of a small tile: there are registers for it)
  const int r = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
  const float start_ratio = w.ratio[batch];
  constexpr bool kEarly = WHAT == kPoly && BM == 64;
  Pack<_Float16, 4> early[2][kEarly ? MI : 1][kEarly ? NJ : 1];
  auto gram_at = [&](int i, int j, int plane) {  // (rows are padded to 64: whole packs)
    const int m = wm + i * 16 + r, n = wn + j * 16 + g * 4;
    return m < rows && n < cols ? load_pack<_Float16, 4>(w.gram + (batch * h.s + m0 + m) * 2 * h.sp + pair_at(n0 + n, plane)) : Pack<_Float16, 4>{};
  };
  if constexpr (kEarly)
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) early[0][i][j] = gram_at(i, j, 0), early[1][i][j] = gram_at(i, j, 1);
  if constexpr (PART != kJoin) {
    __builtin_assume(first < end);  // (no way past the loop to prepare for: 3 x 385 x 129 124 -> 121 us)
#pragma unroll
    for (int i = 0; i < kStages - kGroup; ++i) load(first + i);
    for (int i = first; i < end; i += kGroup) {
      tile_barrier<(kStages - 2 * kGroup) * kLoads>();
#pragma unroll
      for (int u = 0; u < kGroup; ++u) load(i + u + kStages - kGroup);  // (where the stages before i were; zeros behind the last)
#pragma unroll
      for (int u = 0; u < kGroup; ++u) {
        const char* t = lds + (i + u) % kStages * kStage;
        u32x4 fa[2][MI], fb[2][NJ];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            const int n = wn + j * 16;
            fb[p][j] = kSymmetric ? decltype(sb.tile)::fragment(t + BM * kTileRowBytes, n, p)
                                  : decltype(sb.tile)::fragment(t + BM * kTileRowBytes, (int)pair_at(n, p), 0);
          }
#pragma unroll
          for (int q = 0; q < MI; ++q) fa[p][q] = decltype(sa.tile)::fragment(t, wm + q * 16, p);
        }
#pragma unroll
        for (int q = 0; q < MI; ++q)
#pragma unroll
          for (int j = 0; j < NJ; ++j) {
            acc[q][j] = mma_block<_Float16>(fa[0][q], fb[0][j], acc[q][j]);
            fine[q][j] = mma_block<_Float16>(fa[0][q], fb[1][j], fine[q][j]);
            fine[q][j] = mma_block<_Float16>(fa[1][q], fb[0][j], fine[q][j]);
          }
      }
    }
  }
  if constexpr (PART == kShare) {
    f32x4* mine = w.shares + ((int64_t)(part * batches + batch) * tiles + place % tiles) * (NT * MI * NJ) + threadIdx.x;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) mine[(i * NJ + j) * NT] = acc[i][j] + fine[i][j] * kLowUnit;
    tile_barrier<0>();  // (no load is left on its way into LDS)
    return;
  }
  if constexpr (PART == kJoin) {
    const f32x4* from = w.shares + (batch * tiles + place % tiles) * (NT * MI * NJ) + threadIdx.x;
    for (int q = 0; q < parts; ++q, from += (int64_t)batches * tiles * (NT * MI * NJ))
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] += from[(i * NJ + j) * NT];
  }
  tile_barrier<0>();  // (no load is left on its way into LDS)
  const float ratio = ratio_at(start_ratio, step, c.grow);
  // kPoly: a + b r^2 S^ + c r^4 S^ S^ with the coefficients as pairs of floats: an error of a coefficient would be common to all entries and
  // grow like a singular value's | kApply: over the step's growth of r | kLast: X = r X^
  const double r2 = (double)ratio * ratio, cb = c.b * r2 / kScaleS, cc = c.c * r2 * r2 / (kScaleS * kScaleS);
  const float cb_hi = (float)cb, cb_lo = (float)(cb - cb_hi), cc_hi = (float)cc, cc_lo = (float)(cc - cc_hi);
  const float ca_hi = (float)c.a, ca_lo = (float)(c.a - ca_hi);
  // of the sums: to the planes of the result, or to the result itself
  const float out_scale = WHAT == kGram    ? kScaleS / (kScaleX * kScaleX)
                          : WHAT == kApply ? 1.0f / kScaleP * (ratio > 0.0f ? ratio / ratio_at(ratio, 1, c.grow) : 1.0f)
                                           : 1.0f / (kScaleP * kScaleX) * ratio;
  if constexpr (WHAT == kLast) {
    const int image = (h.tall ? BM : BN) * 4;  // bytes of a row of G's direction
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        const int m = wm + i * 16 + r, n = wn + j * 16 + g * 4;
        const f32x4 v = (acc[i][j] + fine[i][j] * kLowUnit) * out_scale;
        if (h.tall) {
#pragma unroll
          for (int q = 0; q < 4; ++q) *reinterpret_cast<float*>(lds + out_addr(n + q, image, m * 4)) = v[q];
        } else {
          *reinterpret_cast<f32x4*>(lds + out_addr(m, image, n * 4)) = v;
        }
      }
    __syncthreads();
    const int r0 = h.tall ? n0 : m0, c0 = h.tall ? m0 : n0, rn = h.tall ? cols : rows, cn = h.tall ? rows : cols;
    const int64_t base = batch * h.m * h.n + (int64_t)r0 * h.n + c0;
    for (int id = threadIdx.x; id < BM * BN / 4; id += NT) {
      const int row = id / (image / 16), col = id % (image / 16) * 4;
      if (row >= rn || col >= cn) continue;
      const f32x4 v = *reinterpret_cast<const f32x4*>(lds + out_addr(row, image, col * 4));
      const int64_t at = base + (int64_t)row * h.n + col;
      const bool whole = col + 4 <= cn;
      if (res.update) {
        float* p = reinterpret_cast<float*>(res.out) + at;
        if (whole) {
          Pack<float, 4> old = load_any<float, 4>(p);
#pragma unroll
          for (int q = 0; q < 4; ++q) old.v[q] = res.keep * old.v[q] - res.rate * v[q];
          store_any(p, old);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (col + q < cn) p[q] = res.keep * p[q] - res.rate * v[q];
        }
      } else {
        T* p = reinterpret_cast<T*>(res.out) + at;
        if (whole) {
          Pack<T, 4> out;
#pragma unroll
          for (int q = 0; q < 4; ++q) out.v[q] = from_f32<T>(v[q]);
          store_any(p, out);
        } else {
#pragma unroll
          for (int q = 0; q < 4; ++q)
            if (col + q < cn) p[q] = from_f32<T>(v[q]);
        }
      }
    }
  } else {
    const int ld = kSymmetric ? h.sp : h.lp;
    _Float16* out = (WHAT == kGram ? w.gram : (WHAT == kPoly ? w.poly : w.x[(step + 1) & 1])) + batch * h.s * 2 * ld;
#pragma unroll
    for (int turned = 0; turned < (kSymmetric ? 2 : 1); ++turned) {
      if (turned) __syncthreads();
      const int image = (turned ? BM : BN) * 4;  // bytes of a row
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) {
          const int m = wm + i * 16 + r, n = wn + j * 16 + g * 4;
          Pack<_Float16, 4> hi, lo, gh{}, gl{};
          if constexpr (kEarly)
            gh = early[0][i][j], gl = early[1][i][j];
          else if constexpr (WHAT == kPoly)
            gh = gram_at(i, j, 0), gl = gram_at(i, j, 1);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float sum = fmaf(fine[i][j][q], kLowUnit, acc[i][j][q]);
            if constexpr (WHAT == kPoly) {
              const bool one = m0 + m == n0 + n + q && m < rows;  // (rows and columns of the padding stay zero)
              const float was = fmaf((float)gl.v[q], kLowUnit, (float)gh.v[q]);
              const float small = fmaf(cc_lo, sum, fmaf(cb_lo, was, one ? ca_lo : 0.0f));
              split((fmaf(cb_hi, was, one ? ca_hi : 0.0f) + fmaf(cc_hi, sum, small)) * kScaleP, hi.v[q], lo.v[q]);
            } else {
              split(sum * out_scale, hi.v[q], lo.v[q]);
            }
            if (turned) {
              *reinterpret_cast<_Float16*>(lds + out_addr(n + q, image, (int)pair_at(m, 0) * 2)) = hi.v[q];
              *reinterpret_cast<_Float16*>(lds + out_addr(n + q, image, (int)pair_at(m, 1) * 2)) = lo.v[q];
            }
          }
          if (!turned) {
            store_pack(reinterpret_cast<_Float16*>(lds + out_addr(m, image, (int)pair_at(n, 0) * 2)), hi);
            store_pack(reinterpret_cast<_Float16*>(lds + out_addr(m, image, (int)pair_at(n, 1) * 2)), lo);
          }
        }
      __syncthreads();
      const int r0 = turned ? n0 : m0, c0 = turned ? m0 : n0, rn = turned ? cols : rows;
      for (int id = threadIdx.x; id < BM * BN * 4 / 16; id += NT) {
        const int row = id / (image / 16), chunk = id % (image / 16), col = c0 + (chunk >> 3) * 32;
        if (row >= rn || col >= ld) continue;
        if (kSymmetric) {  // blocks on and below the diagonal as they are, those below turned
          const int low = turned ? col / BN : (r0 + row) / BN, high = turned ? r0 / BN : n0 / BN;
          if (turned ? low <= high : low < high) continue;
        }
        *reinterpret_cast<u32x4*>(out + (int64_t)(r0 + row) * 2 * ld + 2 * c0 + chunk * 8) = *reinterpret_cast<const u32x4*>(lds + out_addr(row, image, chunk * 16));
      }
    }
  }
}

// tiles of a product of ra x rb
int64_t product_tiles(int bm, int ra, int rb, bool symmetric) {
  const int bn = bm == 64 ? 64 : 128;
  const int64_t m = (ra + bm - 1) / bm, n = (rb + bn - 1) / bn;
  if (!symmetric) return m * n;
  int64_t all = 0;
  for (int t = 0; t < m; ++t) all += symmetric_tiles(t, bm / bn, (int)n);
  return all;
}

// How a product is cut: the cheapest of what a step of k of a round of tiles, one per compute unit, takes: .42 us (64 x 64, of which two or more
// share a compute unit; alone .55), .95 (128 x 128) or 1.65 (256 x 128).  All five steps: 2048 x 4096 with tiles of 256 and 128 1236 us, 64 alone
// 1489; 1024 x 1024 with 64 273, with 128 479; 300 x 128 x 128 with 64 269, with 256 499.  Then the parts of k
// of S: as many as two workgroups per compute unit allow, where they save more steps than they and the second launch cost (1024 x 1024,
// 22 of 32 steps saved: 266 -> 278).
struct ProductPlan {
  int tile, parts;
  int64_t tiles;
};
ProductPlan product_plan(Product what, int ra, int rb, int k, int64_t B) {
  const bool gram = what == kGram, symmetric = gram || what == kPoly;
  ProductPlan best{64, 1, 0};
  double best_cost = 1e30;
  for (int tile = 64; tile <= 256; tile *= 2) {
    const int64_t tiles = product_tiles(tile, ra, rb, symmetric), rounds = (tiles * B + kCompute - 1) / kCompute;
    const double cost = tile == 64 ? (rounds > 1 ? 0.42 * (double)rounds : 0.55) : (tile == 128 ? 0.95 : 1.65) * (double)rounds;
    if (cost < best_cost) best_cost = cost, best.tile = tile, best.tiles = tiles;
  }
  if (best.tile == 64 && gram) {
    const int64_t steps = k / kPairK, room = 2 * kCompute / (best.tiles * B), parts = room < steps / 8 ? room : steps / 8;
    if (parts > 1 && steps - steps / parts > 32) best.parts = (int)parts;
  }
  return best;
}

Work work_of(const Shape& h, int64_t B, void* base) {
  Work w;
  const int64_t x_bytes = B * h.s * (int64_t)h.lp * 4, s_bytes = B * h.s * (int64_t)h.sp * 4;
  char* p = (char*)base;
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) & ~(int64_t)255;
    return q;
  };
  const int64_t parts = h.m * h.n / 8192;  // (at least a few thousand elements each)
  w.parts = (int)(parts < 1 ? 1 : (parts > kNormParts ? kNormParts : parts));
  w.norms = (double*)take(B * kNormParts * 8);
  w.ratio = (float*)take(B * 4);
  w.x[0] = (_Float16*)take(x_bytes);
  w.x[1] = (_Float16*)take(x_bytes);
  w.gram = (_Float16*)take(s_bytes);
  w.poly = (_Float16*)take(s_bytes);
  const ProductPlan gram = product_plan(kGram, h.s, h.s, h.lp, B);
  w.shares = (f32x4*)take(gram.parts > 1 ? gram.parts * gram.tiles * B * 64 * 64 * 4 : 0);
  w.bytes = p - (char*)base;
  return w;
}

template <typename T, Product WHAT, int BM, Part PART>
void launch_product_tile(const ProductPlan& p, const Operands& o, const Shape& h, const Work& w, int64_t B, int step, const Poly& c, const Result& res,
                         hipStream_t s) {
  const int64_t blocks = xcd_blocks(p.tiles * B * (PART == kShare ? p.parts : 1));
  hipFuncSetAttribute((const void*)ns_product_kernel<T, WHAT, BM, PART>, hipFuncAttributeMaxDynamicSharedMemorySize, PairTile<BM>::kLds);
  ns_product_kernel<T, WHAT, BM, PART>
      <<<(unsigned)blocks, PairTile<BM>::kThreads, PairTile<BM>::kLds, s>>>(o, h, w, (int)B, (int)p.tiles, p.parts, step, c, res);
}

template <typename T, Product WHAT>
void launch_product(const Operands& o, const Shape& h, const Work& w, int64_t B, int step, const Poly& c, const Result& res, hipStream_t s) {
  const ProductPlan p = product_plan(WHAT, o.ra, o.rb, o.k, B);
  if constexpr (WHAT == kGram)
    if (p.parts > 1) {
      launch_product_tile<T, WHAT, 64, kShare>(p, o, h, w, B, step, c, res, s);
      return launch_product_tile<T, WHAT, 64, kJoin>(p, o, h, w, B, step, c, res, s);
    }
  if (p.tile == 256) return launch_product_tile<T, WHAT, 256, kAllOfK>(p, o, h, w, B, step, c, res, s);
  if (p.tile == 128) return launch_product_tile<T, WHAT, 128, kAllOfK>(p, o, h, w, B, step, c, res, s);
  return launch_product_tile<T, WHAT, 64, kAllOfK>(p, o, h, w, B, step, c, res, s);
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix whose short side fits four 16-row blocks stays in one workgroup's LDS from the first read to the last write: fp32 throughout,
// products on the fp32 matrix instructions, which at these sizes wait for the LDS rather than for each other, and ONE launch for every
// small matrix of a whole list of stacks, where the planes' path needs three launches a step.  Eight waves: a wave takes two of the (up to)
// 16 blocks of S and of P, and half the rows of a 16-column block of X.
// 80 matrices of 64 x 64 and smaller in five stacks, momentum and parameters included: 36 us, five steps of three products each behind the
// one before it in the same LDS.
// LDS rows are 64 i + 4 floats apart: 16 rows x 4 k (chunk reads of A and B) and 4 k x 16 columns (the reads of X as B) both meet all 64
// banks once.
constexpr int kSmallSide = 64;
constexpr int kSmallLds = 150 * 1024;
constexpr int kSmallThreads = 512;
constexpr int kSmallMax = 24;  // stacks per launch
constexpr int kSmallLd = kSmallSide + 4;

struct SmallStack {
  Source src;
  Result res;
  int first;  // first workgroup
  int m, n;
};
struct SmallStacks {
  int count;
  SmallStack stack[kSmallMax];
};

__host__ __device__ inline int round16(int v) { return (v + 15) & ~15; }
__host__ __device__ inline int small_ld(int l) { return ((l + 63) & ~63) + 4; }
inline int64_t small_lds_bytes(int64_t s, int64_t l) { return (round16((int)s) * (int64_t)small_ld((int)l) + 2 * round16((int)s) * kSmallLd) * 4; }
// (a few long ones are better spread over the chip: 32 x 1024 153 us here, 121 there; 256 of 64 x 256 81 and 300)
inline bool is_small(int64_t B, int64_t m, int64_t n) {
  const int64_t s = m < n ? m : n, l = m < n ? n : m;
  return s <= kSmallSide && l <= 4096 && small_lds_bytes(s, l) <= kSmallLds && (l <= 512 || B >= 64);
}

// two 16 x 16 blocks of rows . rows^T: acc[j] = A(16 i .., :) B(16 (j0 + j) .., :)^T over k
__device__ __forceinline__ void small_rows(const float* a, const float* b0, const float* b1, int k, f32x4& acc0, f32x4& acc1) {
  for (int t = 0; t < k; t += 16) {
    const f32x4 av = *reinterpret_cast<const f32x4*>(a + t), bv0 = *reinterpret_cast<const f32x4*>(b0 + t), bv1 = *reinterpret_cast<const f32x4*>(b1 + t);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      acc0 = __builtin_amdgcn_mfma_f32_16x16x4f32(av[q], bv0[q], acc0, 0, 0, 0);
      acc1 = __builtin_amdgcn_mfma_f32_16x16x4f32(av[q], bv1[q], acc1, 0, 0, 0);
    }
  }
}

template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(kSmallThreads) void ns_small_kernel(SmallStacks all, int steps, Poly c, float eps) {
  extern __shared__ __attribute__((aligned(16))) float sm[];
  __shared__ double part[kSmallThreads / 64];
  int which = 0;
  while (which + 1 < all.count && (int)blockIdx.x >= all.stack[which + 1].first) ++which;
  const SmallStack& st = all.stack[which];
  const int m = st.m, n = st.n, size = m * n;
  const bool tall = m > n;
  const int s = tall ? n : m, l = tall ? m : n, sr = round16(s), lr = round16(l), ld = small_ld(l), nb = sr / 16;
  float* X = sm;
  float* S = X + sr * ld;
  float* P = S + sr * kSmallLd;
  const int64_t base = (int64_t)((int)blockIdx.x - st.first) * size;
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, r = lane & 15, g = lane >> 4;
  double sum = 0.0;
  for (int i = threadIdx.x; i < sr * lr; i += kSmallThreads) {  // (the padding)
    const int row = i / lr, col = i - row * lr;
    if (row >= s || col >= l) X[row * ld + col] = 0.0f;
  }
  for (int i = threadIdx.x; i < size; i += kSmallThreads) {
    const float v = source_value<T, MOMENTUM, true>(st.src, base + i);
    const int row = i / n, col = i - row * n;
    X[tall ? col * ld + row : row * ld + col] = v;
    sum += (double)v * v;
  }
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if (lane == 0) part[wave] = sum;
  __syncthreads();
  sum = 0.0;
  for (int i = 0; i < kSmallThreads / 64; ++i) sum += part[i];
  const double norm = sqrt(sum), inv = norm == 0.0 ? 0.0 : 1.0 / (norm + (double)eps);
  for (int i = threadIdx.x; i < s * l; i += kSmallThreads) {
    const int row = i / l, at = row * ld + i - row * l;
    X[at] = (float)(X[at] * inv);
  }
  __syncthreads();
  const int bi = wave >> 1, bj = (wave & 1) * 2;  // this wave's blocks of S and P: (bi, bj), (bi, bj + 1)
  const bool mine = bi < nb && bj < nb, two = mine && bj + 1 < nb;
  const int units = 2 * (lr / 16);  // halves of column blocks of X
  for (int step = 0; step < steps; ++step) {
    f32x4 acc[2];
    const f32x4 zero = {0.f, 0.f, 0.f, 0.f};
    if (mine) {
      acc[0] = acc[1] = zero;
      const float* b0 = X + (bj * 16 + r) * ld + 4 * g;
      small_rows(X + (bi * 16 + r) * ld + 4 * g, b0, two ? b0 + 16 * ld : b0, lr, acc[0], acc[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j == 0 || two)
#pragma unroll
          for (int q = 0; q < 4; ++q) S[(bi * 16 + 4 * g + q) * kSmallLd + (bj + j) * 16 + r] = acc[j][q];
    }
    __syncthreads();
    if (mine) {
      acc[0] = acc[1] = zero;
      const float* b0 = S + (bj * 16 + r) * kSmallLd + 4 * g;
      small_rows(S + (bi * 16 + r) * kSmallLd + 4 * g, b0, two ? b0 + 16 * kSmallLd : b0, sr, acc[0], acc[1]);
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j == 0 || two)
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const int row = bi * 16 + 4 * g + q, col = (bj + j) * 16 + r, at = row * kSmallLd + col;
            P[at] = (float)(c.c * acc[j][q] + (c.b * S[at] + (row == col ? c.a : 0.0)));
          }
    }
    __syncthreads();
    for (int u0 = 0; u0 < units; u0 += kSmallThreads / 64) {
      const int u = u0 + wave, col = (u >> 1) * 16 + r, i0 = (u & 1) * 2;
      const bool on = u < units && i0 < nb, both = on && i0 + 1 < nb;
      acc[0] = acc[1] = zero;
      if (on) {
        const float* a0 = P + (i0 * 16 + r) * kSmallLd + 4 * g;
        const float* a1 = both ? a0 + 16 * kSmallLd : a0;
        const float* b = X + 4 * g * ld + col;
        for (int t = 0; t < sr; t += 16) {
          const f32x4 av0 = *reinterpret_cast<const f32x4*>(a0 + t), av1 = *reinterpret_cast<const f32x4*>(a1 + t);
#pragma unroll
          for (int q = 0; q < 4; ++q) {
            const float bv = b[(t + q) * ld];
            acc[0] = __builtin_amdgcn_mfma_f32_16x16x4f32(av0[q], bv, acc[0], 0, 0, 0);
            acc[1] = __builtin_amdgcn_mfma_f32_16x16x4f32(av1[q], bv, acc[1], 0, 0, 0);
          }
        }
      }
      __syncthreads();  // (both halves of a column block have read it)
#pragma unroll
      for (int j = 0; j < 2; ++j)
        if (j == 0 ? on : both)
#pragma unroll
          for (int q = 0; q < 4; ++q) X[((i0 + j) * 16 + 4 * g + q) * ld + col] = acc[j][q];
    }
    __syncthreads();
  }
  for (int i = threadIdx.x; i < size; i += kSmallThreads) {
    const int row = i / n, col = i - row * n;
    const float v = X[tall ? col * ld + row : row * ld + col];
    if (st.res.update) {
      float* p = reinterpret_cast<float*>(st.res.out) + base + i;
      *p = st.res.keep * *p - st.res.rate * v;
    } else {
      reinterpret_cast<T*>(st.res.out)[base + i] = from_f32<T>(v);
    }
  }
}

template <typename T, bool MOMENTUM>
void launch_small(const SmallStacks& all, int blocks, int64_t lds, int steps, const Poly& c, float eps, hipStream_t s) {
  if (lds > 64 * 1024) hipFuncSetAttribute((const void*)ns_small_kernel<T, MOMENTUM>, hipFuncAttributeMaxDynamicSharedMemorySize, kSmallLds);
  ns_small_kernel<T, MOMENTUM><<<(unsigned)blocks, kSmallThreads, (size_t)lds, s>>>(all, steps, c, eps);
}

template <typename T, bool MOMENTUM>
int run(const Source& src, int64_t B, int64_t m, int64_t n, int steps, const Poly& c, float eps, const Result& res, void* workspace, hipStream_t s) {
  if (is_small(B, m, n)) {
    SmallStacks one;
    one.count = 1;
    one.stack[0] = {src, res, 0, (int)m, (int)n};
    launch_small<T, MOMENTUM>(one, (int)B, small_lds_bytes(m < n ? m : n, m < n ? n : m), steps, c, eps, s);
    PS_CHECK_LAUNCH();
  }
  const Shape h = shape_of(m, n);
  const Work w = work_of(h, B, workspace);
  const dim3 norm_grid((unsigned)w.parts, (unsigned)B);
  const dim3 start_grid((unsigned)((h.tall ? h.sp : h.lp) / 64), (unsigned)((h.tall ? h.lp : h.sp) / 64), (unsigned)B);
  ns_norm_kernel<T, MOMENTUM><<<norm_grid, 256, 0, s>>>(src, m * n, w);
  ns_start_kernel<T, MOMENTUM><<<start_grid, 256, 0, s>>>(src, h, w, eps);
  for (int i = 0; i < steps; ++i) {
    const _Float16* x = w.x[i & 1];
    launch_product<float, kGram>({x, x, h.s, h.s, h.lp, 0, 0}, h, w, B, i, c, res, s);
    launch_product<float, kPoly>({w.gram, w.gram, h.s, h.s, h.sp, 0, 0}, h, w, B, i, c, res, s);
    const Operands apply{w.poly, x, h.s, h.l, h.sp, h.s, h.lp};
    if (i + 1 < steps)
      launch_product<float, kApply>(apply, h, w, B, i, c, res, s);
    else
      launch_product<T, kLast>(apply, h, w, B, i, c, res, s);
  }
  PS_CHECK_LAUNCH();
}

constexpr int64_t kMaxSide = 1 << 20;

bool sizes_ok(int64_t B, int64_t m, int64_t n, int steps) {
  return B >= 0 && B <= 65535 && m >= 0 && n >= 0 && m <= kMaxSide && n <= kMaxSide && steps >= 1 && steps <= 64 && (m < n ? m : n) <= 16384 &&
         ((m + 63) / 64) * ((n + 63) / 64) * B < kMaxThreads / 256 - kXcds;  // (tiles of 64 x 64: the most threads a launch takes)
}

}  // namespace

extern "C" int64_t ps_newton_schulz_workspace(int64_t B, int64_t m, int64_t n) {
  if (!sizes_ok(B, m, n, 1) || B == 0 || m == 0 || n == 0 || is_small(B, m, n)) return 0;
  return work_of(shape_of(m, n), B, nullptr).bytes;
}

extern "C" int ps_newton_schulz(const void* g, int64_t B, int64_t m, int64_t n, int dtype, int steps, double a, double b, double c, float grow, float eps, void* out,
                                void* workspace, void* stream) {
  PS_REQUIRE(sizes_ok(B, m, n, steps) && grow >= 1.0f, "ps_newton_schulz: sizes out of range");
  if (B == 0 || m == 0 || n == 0) return 0;
  PS_REQUIRE(g != nullptr && out != nullptr && (workspace != nullptr || is_small(B, m, n)), "ps_newton_schulz: null argument");
  const Poly co{a, b, c, grow};
  const Source src{g, nullptr, 0.0f, 1.0f, 0};
  const Result res{out, 0, 0.0f, 0.0f};
  if (dtype == kF32) return run<float, false>(src, B, m, n, steps, co, eps, res, workspace, (hipStream_t)stream);
  if (dtype == kF16) return run<_Float16, false>(src, B, m, n, steps, co, eps, res, workspace, (hipStream_t)stream);
  if (dtype == kBF16) return run<__bf16, false>(src, B, m, n, steps, co, eps, res, workspace, (hipStream_t)stream);
  ps_set_error("ps_newton_schulz: unknown element type (0 fp32, 1 fp16, 2 bf16)");
  return -1;
}

// n_stacks stacks of parameters, every argument with an index a HOST array; the small matrices of all of them go out together
extern "C" int ps_muon_step(int n_stacks, float* const* p, const float* const* g, float* const* buf, const int64_t* B, const int64_t* m, const int64_t* n,
                            const float* rate, double momentum, int nesterov, float keep, int steps, double a, double b, double c, float grow,
                            float eps, void* workspace, void* stream) {
  PS_REQUIRE(n_stacks >= 0 && grow >= 1.0f, "ps_muon_step: sizes out of range");
  PS_REQUIRE(n_stacks == 0 || (p && g && buf && B && m && n && rate), "ps_muon_step: null argument");
  for (int i = 0; i < n_stacks; ++i) {
    PS_REQUIRE(sizes_ok(B[i], m[i], n[i], steps), "ps_muon_step: sizes out of range");
    PS_REQUIRE(B[i] * m[i] * n[i] == 0 || (p[i] && g[i] && buf[i] && (workspace || is_small(B[i], m[i], n[i]))), "ps_muon_step: null argument");
  }
  const Poly co{a, b, c, grow};
  hipStream_t s = (hipStream_t)stream;
  SmallStacks all;
  all.count = 0;
  int blocks = 0;
  int64_t lds = 0;
  auto flush = [&] {
    if (all.count > 0) launch_small<float, true>(all, blocks, lds, steps, co, eps, s);
    all.count = blocks = 0;
    lds = 0;
  };
  for (int i = 0; i < n_stacks; ++i) {
    if (B[i] == 0 || m[i] == 0 || n[i] == 0) continue;
    const Source src{g[i], buf[i], (float)momentum, (float)(1.0 - momentum), nesterov};
    const Result res{p[i], 1, keep, rate[i]};
    if (!is_small(B[i], m[i], n[i])) {
      const int rc = run<float, true>(src, B[i], m[i], n[i], steps, co, eps, res, workspace, s);
      if (rc != 0) return rc;
      continue;
    }
    const int64_t need = small_lds_bytes(m[i] < n[i] ? m[i] : n[i], m[i] < n[i] ? n[i] : m[i]);
    all.stack[all.count++] = {src, res, blocks, (int)m[i], (int)n[i]};
    blocks += (int)B[i];
    lds = need > lds ? need : lds;
    if (all.count == kSmallMax) flush();
  }
  flush();
  PS_CHECK_LAUNCH();
}
