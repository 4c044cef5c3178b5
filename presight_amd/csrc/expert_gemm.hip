// The experts' linear layers on rows sorted by expert: rows [M, in], offsets [E+1] (expert e's rows are offsets[e] .. offsets[e+1]),
// weight [E, out, in], bias [E, out].
//     y[p]  = W_e x[p] + b_e                     tiles of (rows of one expert) x (out),  k = in     x k-contiguous, W k-contiguous
//     dx[p] = W_e^T dy[p]                        tiles of (rows of one expert) x (in),   k = out    dy k-contiguous, W row-contiguous
//     dW_e  = sum_p dy[p] x[p]^T, db_e = sum_p dy[p]   tiles of (out) x (in) of one expert, k = its rows, both row-contiguous
// The experts' lengths are known on the device only.  A launch holds ceil(M / BM) + E row tiles and one workgroup more, which is enough for
// any split of the rows; every workgroup finds its expert and tile from the offsets, and those left over clear the rows of nobody.
#include <type_traits>
#include "gemm_core.hpp"

namespace {

using namespace ps;

struct RowTile {
  int expert;
  int64_t row0;  // first row of the tile
  int rows;      // rows of the tile
};

__device__ __forceinline__ int64_t bounded(int v, int64_t M) { return v < 0 ? 0 : (v > M ? M : v); }

// what M rows of E experts can make at most
__host__ __device__ inline int64_t row_tiles_at_most(int64_t M, int E, int piece) { return (M + piece - 1) / piece + (M < E ? M : E); }

// ... and those of more than `above` rows: one piece more than its share for each, of M / (above + 1) at most
__host__ __device__ inline int64_t crowded_pieces_at_most(int64_t M, int above) { return 2 * (M / above); }

// The tiles of `piece` rows that the experts' rows make (above > 0: pieces of `above` rows, of the experts with more than that): a prefix sum over
// the lanes, each with its share of neighbouring experts, and a second one over the experts of the lane that holds the tile, where it has several.  (64 experts after the other instead, and a workgroup per
// expert whether it can have rows or not: 16 rows of 256 experts, 1024 x 2048 bf16, 30.7 us for 14.9; 8192 of 1024, 256 x 512, 157 for 80.)
struct RowTiles {
  const int* offsets;
  int64_t M;
  int E, piece, above, each;  // each: experts per lane
  int lo, len;         // rows of this lane's last expert
  unsigned mine, incl; // tiles of this lane's experts; up to and with them
  int total;           // tiles in all

  __device__ __forceinline__ unsigned read(int e) {  // -> tiles of expert e
    const int64_t first = bounded(offsets[e], M), end = bounded(offsets[e + 1], M);
    lo = (int)first;
    len = end > first ? (int)(end - first) : 0;
    if (len <= above) len = 0;
    return ((unsigned)len + (unsigned)piece - 1u) / (unsigned)piece;
  }
  __device__ __forceinline__ unsigned scan() {  // incl from mine -> their sum
    incl = mine;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
      const unsigned o = __shfl_up(incl, d, 64);
      if ((int)(threadIdx.x & 63) >= d) incl += o;
    }
    return (unsigned)__builtin_amdgcn_readlane((int)incl, 63);
  }
  __device__ __forceinline__ RowTiles(const int* offsets_, int E_, int64_t M_, int piece_, int above_ = 0)
      : offsets(offsets_), M(M_), E(E_), piece(piece_), above(above_), each((E_ + 63) / 64), lo(0), len(0), mine(0), total(0) {
    // (offsets that do not ascend could ask for more than there is room for; 64 lanes' `most` stay below 2^32)
    const unsigned most = (unsigned)(above > 0 ? crowded_pieces_at_most(M, above) : row_tiles_at_most(M, E, piece));
    const int e0 = (threadIdx.x & 63) * each, e1 = e0 + each < E ? e0 + each : E;
#pragma unroll 4
    for (int e = e0; e < e1; ++e) {
      const unsigned sum = mine + read(e);
      mine = sum < most ? sum : most;
    }
    const unsigned sum = scan();
    total = (int)(sum < most ? sum : most);
  }
  // tile t < total, uniform over the wave
  __device__ __forceinline__ RowTile find(int t_) const {
    RowTiles s = *this;
    unsigned t = (unsigned)t_;
    int who = uniform(__ffsll((long long)__ballot(t < s.incl)) - 1), e0 = 0;
    if (each > 1) {
      t -= (unsigned)__builtin_amdgcn_readlane((int)(s.incl - s.mine), who);
      e0 = who * each;
      const int e1 = e0 + each < E ? e0 + each : E;
      for (;; e0 += 64) {
        const int e = e0 + (threadIdx.x & 63);
        s.mine = e < e1 ? s.read(e) : 0;
        const unsigned n = s.scan();
        if (t < n || e0 + 64 >= e1) break;
        t -= n;
      }
      who = uniform(__ffsll((long long)__ballot(t < s.incl)) - 1);
    }
    const int n = __builtin_amdgcn_readlane(s.len, who), k = (int)(t - (unsigned)__builtin_amdgcn_readlane((int)(s.incl - s.mine), who));
    return {e0 + who, (int64_t)__builtin_amdgcn_readlane(s.lo, who) + (int64_t)k * piece, n - k * piece < piece ? n - k * piece : piece};
  }
};

// zeros to the rows before offsets[0] and from offsets[E] on, shared out over `many` workgroups
template <typename T>
__device__ __forceinline__ void clear_outside(const int* __restrict__ offsets, int E, int64_t M, int me, int many, T* __restrict__ y, int N) {
  const int64_t head = bounded(offsets[0], M), end = bounded(offsets[E], M), tail0 = end > head ? end : head;
  const int64_t count = (head + (M - tail0)) * N, step = (int64_t)many * blockDim.x;
  const int64_t first = head * N;
  for (int64_t i = (int64_t)me * blockDim.x + threadIdx.x; i < count; i += step) y[i < first ? i : tail0 * N + (i - first)] = from_f32<T>(0.0f);
}

// Two stages of 128 bytes of k in LDS: the loads of the next tile are in flight while the matrix instructions run over this one.  What a
// compute unit can have in flight from the L2 bounds them (about 18 bytes a cycle): a 256 x 256 tile of 16-bit operands asks for 32 at the
// full matrix rate, a 128 x 128 one for 64.  (8192 x 8192 x 8192 bf16: 859 us, 1281 TFLOP/s; four stages of half the depth, half a tile of
// fragments read ahead, and several tiles per workgroup with the next one's loads under this one's store were no faster.)
// SUMS: also the sums of A's rows over k, as a product with ones (`sums`: whether this wave wants them).
template <typename T, int BM, int BN, int WM, int WN, bool A_RC, bool B_RC, bool SUMS>
__device__ __forceinline__ void direct_loop(char* lds, int K, const DirectSource<T, BM, 64 * WM * WN, A_RC>& sa,
                                            const DirectSource<T, BN, 64 * WM * WN, B_RC>& sb, f32x4 (&acc)[BM / WM / 16][BN / WN / 16],
                                            f32x4 (&row_sums)[SUMS ? BM / WM / 16 : 1], bool sums) {
  constexpr int MI = BM / WM / 16, NJ = BN / WN / 16, BK = kTileK<T>, kStage = (BM + BN) * kTileRowBytes;
  using TA = DirectTile<T, BM, 64 * WM * WN, A_RC>;
  using TB = DirectTile<T, BN, 64 * WM * WN, B_RC>;
  const int wave = threadIdx.x >> 6, wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  u32x4 ones;
  if constexpr (SUMS) {
    const unsigned one = sizeof(T) == 4 ? 0x3f800000u : (__is_same(T, _Float16) ? 0x3c003c00u : 0x3f803f80u);
    ones = u32x4{one, one, one, one};
#pragma unroll
    for (int i = 0; i < MI; ++i) row_sums[i] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  if (K <= 0) return;
  sa.load(0, lds);
  sb.load(0, lds + BM * kTileRowBytes);
  tile_barrier<0>();
  for (int k0 = 0, cur = 0; k0 < K; k0 += BK, cur ^= 1) {
    char* a = lds + cur * kStage;
    if (k0 + BK < K) {
      char* next = lds + (cur ^ 1) * kStage;
      sa.load(k0 + BK, next);
      sb.load(k0 + BK, next + BM * kTileRowBytes);
    }
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u32x4 fa[MI], fb[NJ];
#pragma unroll
      for (int i = 0; i < MI; ++i) fa[i] = TA::fragment(a, wm + i * 16, s);
#pragma unroll
      for (int j = 0; j < NJ; ++j) fb[j] = TB::fragment(a + BM * kTileRowBytes, wn + j * 16, s);
#pragma unroll
      for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NJ; ++j) acc[i][j] = mma_block<T>(fa[i], fb[j], acc[i][j]);
      if constexpr (SUMS) {
        if (sums)
#pragma unroll
          for (int i = 0; i < MI; ++i) row_sums[i] = mma_block<T>(fa[i], ones, row_sums[i]);
      }
    }
    tile_barrier<0>();
  }
}

// A wave's part of a tile into memory, turned in LDS on the way: four values per lane and row make requests of 8 to 16 bytes (65536 x
// 1024 bf16: 12.6 million of them, a third of the kernel's time); from a row of the wave's own LDS slice (MI * 16 rows in as many passes
// as it takes) every lane writes 16 bytes of whole 64- to 256-byte rows.  No other wave reads the slice, and the tiles are done with.
template <typename T, int MI, int NJ, int SLICE, typename Bias>
__device__ __forceinline__ void store_tile_rows(f32x4 (&acc)[MI][NJ], char* slice, T* __restrict__ y, int64_t ldy, int rows, int cols, int m0, int n0,
                                                const Bias* __restrict__ bias) {
  constexpr int kRow = NJ * 16 * (int)sizeof(T), kAcross = kRow / 16;  // bytes and chunks of a row
  constexpr int kFit = SLICE / (16 * kRow), kPass = kFit < MI ? kFit : MI;  // blocks of 16 rows per pass
  constexpr int kSpread = kAcross < 8 ? kAcross - 1 : 7;
  static_assert(kPass >= 1 && MI % kPass == 0, "whole blocks of rows per pass");
  const int lane = threadIdx.x & 63, r = lane & 15, g = lane >> 4;
  float b[NJ][4] = {};
  if (bias != nullptr) {
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + j * 16 + g * 4 + q;
        if (n < cols) b[j][q] = to_f32(bias[n]);
      }
  }
#pragma unroll
  for (int p = 0; p < MI / kPass; ++p) {
#pragma unroll
    for (int i = 0; i < kPass; ++i)
#pragma unroll
      for (int j = 0; j < NJ; ++j) {
        Pack<T, 4> o;
#pragma unroll
        for (int q = 0; q < 4; ++q) o.v[q] = from_f32<T>(acc[p * kPass + i][j][q] + b[j][q]);
        const int row = i * 16 + r, byte = (j * 16 + g * 4) * (int)sizeof(T);
        store_pack(reinterpret_cast<T*>(slice + row * kRow + (((byte >> 4) ^ (row & kSpread)) << 4) + (byte & 15)), o);
      }
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
    for (int t = 0; t < kPass * 16 * kAcross / 64; ++t) {
      const int id = t * 64 + lane, row = id / kAcross, c = id % kAcross, m = m0 + p * kPass * 16 + row, n = n0 + c * kChunk<T>;
      const u32x4 v = *reinterpret_cast<const u32x4*>(slice + row * kRow + ((c ^ (row & kSpread)) << 4));
      if (m >= rows || n >= cols) continue;
      T* p = y + m * ldy + n;
      const auto pack = __builtin_bit_cast(Pack<T, kChunk<T>>, v);
      if (n + kChunk<T> <= cols) {
        store_any(p, pack);
      } else {
#pragma unroll
        for (int q = 0; q < kChunk<T>; ++q)
          if (n + q < cols) p[q] = pack.v[q];
      }
    }
    __builtin_amdgcn_wave_barrier();
  }
}

// What bounds it depends on the rows per expert.  16 rows of 16 experts' 1024 x 2048 bf16: the weights' 67 MB, 13.4 us, 5.0 TB/s.  131072 rows of 64
// fp32, 16 experts: the rows' 67 MB and the launch, 21 us.  65536 rows, 2048 x 1024 bf16, 32 experts: the compute units' reads from the
// L2 and the power limit (a tenth less time on zeros), and the experts' last, incomplete tiles: 302 us forward, 310 for the input gradient, 910 and
// 887 TFLOP/s; 286 and 295 where every expert has 2048 rows.  (Those tiles in a round of their own behind the whole ones, and lines fetched into
// the L2 two to eight steps of k ahead, were slower.)
// y[p] = sum_k x[p][k] W(n,k) (+ bias).  W_RC = false: the weight's rows are k-contiguous (forward), n of them; true: n-contiguous (input
// gradient), `w_rows` of them.  K: the rows' length in whole chunks.
// SHARED: k is shared out over `parts` workgroups per tile, whose fp32 sums go to y [parts][M][N]; linear_join_kernel adds them up in order.
template <typename T, int BM, int BN, int WM, int WN, bool W_RC, bool SHARED>
__global__ __launch_bounds__(64 * WM * WN) void linear_kernel(const T* __restrict__ x, int64_t ldx, const T* __restrict__ weight, int64_t ldw, int w_rows,
                                                              const T* __restrict__ bias, const int* __restrict__ offsets, int64_t M, int E, int N, int K,
                                                              int parts, std::conditional_t<SHARED, float, T>* __restrict__ y) {
  constexpr int NT = 64 * WM * WN, MI = BM / WM / 16, NJ = BN / WN / 16;
  using Out = std::conditional_t<SHARED, float, T>;
  int k_rows = w_rows;  // of a weight with k along its rows
  extern __shared__ __attribute__((aligned(16))) char lds[];
  RowTiles tiles(offsets, E, M, BM);
  const int n_tiles = (N + BN - 1) / BN, all = tiles.total * n_tiles;
  int place = xcd_place(blockIdx.x, SHARED ? all * parts : all);
  if (place < 0) {
    if constexpr (!SHARED) clear_outside<T>(offsets, E, M, xcd_spare(blockIdx.x, gridDim.x, all), gridDim.x - all, y, N);
    return;
  }
  if constexpr (SHARED) {
    const int part = place / all, steps = (K + kTileK<T> - 1) / kTileK<T>;
    const int k0 = (int)((int64_t)steps * part / parts) * kTileK<T>, k1 = (int)((int64_t)steps * (part + 1) / parts) * kTileK<T>;
    place -= part * all;
    y += (int64_t)part * M * N;
    x += k0;
    weight += W_RC ? k0 * ldw : k0;
    k_rows = w_rows - k0 < k1 - k0 ? w_rows - k0 : k1 - k0;
    K = (k1 < K ? k1 : K) - k0;
    if (part > 0) bias = nullptr;
  }
  const TileAt at = patched_tile(place, tiles.total, n_tiles);
  const RowTile t = tiles.find(at.m);
  const int n0 = at.n * BN, cols = N - n0 < BN ? N - n0 : BN;
  const T* wb = weight + (int64_t)t.expert * w_rows * ldw + (W_RC ? (int64_t)n0 : n0 * ldw);
  const DirectSource<T, BM, NT, false> sa(x + t.row0 * ldx, ldx, t.rows, K);
  const DirectSource<T, BN, NT, W_RC> sb(wb, ldw, W_RC ? (N + kChunk<T> - 1) / kChunk<T> * kChunk<T> - n0 : cols, W_RC ? k_rows : K);
  f32x4 acc[MI][NJ], none[1];
  direct_loop<T, BM, BN, WM, WN, false, W_RC, false>(lds, K, sa, sb, acc, none, false);
  const int wave = uniform(threadIdx.x >> 6), wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  constexpr int kSlice = 2 * (BM + BN) * kTileRowBytes / (WM * WN);
  store_tile_rows<Out, MI, NJ, kSlice>(acc, lds + wave * kSlice, y + t.row0 * N + n0, N, t.rows, cols, wm, wn,
                                       bias != nullptr ? bias + (int64_t)t.expert * N + n0 : nullptr);
}

// y [M,N] = the sums of parts [parts][M][N]; zeros for the rows of nobody
template <typename T>
__global__ __launch_bounds__(256) void linear_join_kernel(const float* __restrict__ sums, int parts, const int* __restrict__ offsets, int E, int64_t M, int N,
                                                          T* __restrict__ y) {
  const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x, row = i / N, size = M * N;
  if (i >= size) return;
  float v = 0.0f;
  if (row >= bounded(offsets[0], M) && row < bounded(offsets[E], M))
#pragma unroll 4
    for (int p = 0; p < parts; ++p) v += sums[p * size + i];
  y[i] = from_f32<T>(v);
}

// Weight gradients.  Few and small weights with many rows would leave most of the chip idle: then (SPLIT) the experts' rows are cut into
// pieces of `piece` rows, whoever they belong to, every piece writes its own fp32 sums [unit][out][in] (and [unit][out]), and
// dw_join_kernel adds up the pieces of each expert in order.  Also shorter sums: a piece rounds `piece` / 4 times where the whole
// column would round a hundred times as often.
// 65536 rows, 2048 x 1024 bf16, 32 experts (whole): 258 us, 1065 TFLOP/s; 131072 rows of 64 x 64 fp32, 16 experts (pieces): 21 us and 5 to join.
// Many experts whose share is short are summed whole, but all rows may go to a few of them (kCrowded): the first `piece_blocks` workgroups take the
// pieces of those with more than `piece` rows, the others leave these experts out, and dw_join_crowded_kernel adds the pieces up.
enum DwCut { kWhole, kPieces, kCrowded };

template <typename T, int BM, int BN, int WM, int WN, DwCut CUT>
__global__ __launch_bounds__(64 * WM * WN) void linear_dw_kernel(const T* __restrict__ dy, int64_t ldy, const T* __restrict__ x, int64_t ldx,
                                                                 const int* __restrict__ offsets, int64_t M, int E, int N, int K, int ldo, int piece,
                                                                 int piece_blocks, void* __restrict__ dw, void* __restrict__ db,
                                                                 float* __restrict__ parts, float* __restrict__ db_parts) {
  constexpr int NT = 64 * WM * WN, MI = BM / WM / 16, NJ = BN / WN / 16;
  extern __shared__ __attribute__((aligned(16))) char lds[];
  const int n_tiles = (K + BN - 1) / BN, m_tiles = (N + BM - 1) / BM;
  // (a unit's tiles share all of their operands: they stay on one XCD)
  const int tiles = n_tiles * m_tiles;
  const bool cut = CUT == kPieces || (CUT == kCrowded && (int)blockIdx.x < piece_blocks);
  int units = E, unit, len;
  int64_t row0;
  RowTiles pieces(offsets, cut ? E : 0, M, CUT == kWhole ? 1 : piece, CUT == kCrowded ? piece : 0);
  if (cut) units = pieces.total;
  const int place = xcd_place(CUT == kCrowded && !cut ? (int)blockIdx.x - piece_blocks : (int)blockIdx.x, units * tiles);
  if (place < 0) return;
  unit = place / tiles;
  const int tn = place % n_tiles, tm = place % tiles / n_tiles;
  if (cut) {
    const RowTile t = pieces.find(unit);
    row0 = t.row0;
    len = t.rows;
  } else {
    const int64_t lo = bounded(offsets[unit], M), hi = bounded(offsets[unit + 1], M);
    row0 = lo;
    len = uniform(hi > lo ? (int)(hi - lo) : 0);
    if (CUT == kCrowded && len > piece) return;
  }
  const int m0 = tm * BM, n0 = tn * BN;
  constexpr int kC = kChunk<T>;  // (rows hold whole chunks)
  const DirectSource<T, BM, NT, true> sa(dy + row0 * ldy + m0, ldy, (N + kC - 1) / kC * kC - m0, len);
  const DirectSource<T, BN, NT, true> sb(x + row0 * ldx + n0, ldx, (K + kC - 1) / kC * kC - n0, len);
  const int wave = uniform(threadIdx.x >> 6), wm = (wave / WN) * (BM / WM), wn = (wave % WN) * (BN / WN);
  const bool sums = db != nullptr && tn == 0 && wn == 0;
  f32x4 acc[MI][NJ], row_sums[MI];
  direct_loop<T, BM, BN, WM, WN, true, true, true>(lds, len, sa, sb, acc, row_sums, sums);
  constexpr int kSlice = 2 * (BM + BN) * kTileRowBytes / (WM * WN);
  auto leave = [&](auto* o, int64_t ld, auto* ob, int64_t ldb) {
    using Out = std::remove_pointer_t<decltype(o)>;
    store_tile_rows<Out, MI, NJ, kSlice>(acc, lds + wave * kSlice, o + ((int64_t)unit * N + m0) * ld + n0, ld, N - m0 < BM ? N - m0 : BM,
                                         K - n0 < BN ? K - n0 : BN, wm, wn, static_cast<const Out*>(nullptr));
    if (sums && (threadIdx.x & 63) < 16) {
#pragma unroll
      for (int i = 0; i < MI; ++i) {
        const int m = m0 + wm + i * 16 + (threadIdx.x & 15);
        if (m < N) ob[(int64_t)unit * ldb + m] = from_f32<Out>(row_sums[i][0]);
      }
    }
  };
  if (cut)
    leave(parts, ldo, db_parts, (N + 3) / 4 * 4);
  else
    leave(reinterpret_cast<T*>(dw), K, reinterpret_cast<T*>(db), N);
}

// dW_e, db_e = the sums of expert e's n pieces from `first` on: parts [unit][out][ldo] (ldo: in, rounded up to four) and db_parts [unit][out
// rounded up].  Four lanes share the pieces of four neighbouring sums, each takes every fourth in order, and the four meet in LDS in order.
template <typename T>
__device__ __forceinline__ void join_pieces(const float* __restrict__ parts, const float* __restrict__ db_parts, int e, int64_t first, int n, int64_t chunk, int N,
                                            int K, int ldo, T* __restrict__ dw, T* __restrict__ db) {
  __shared__ f32x4 quarter[4][64];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t size = (int64_t)N * ldo, db_size = (N + 3) / 4 * 4, i = (chunk * 64 + lane) * 4;
  const bool bias = i >= size;  // (the weights' sums first, then the bias's)
  const float* p = bias ? db_parts + first * db_size + (i - size) : parts + first * size + i;
  const int64_t step = bias ? db_size : size;
  const bool on = i < size || (db != nullptr && i < size + db_size);
  f32x4 v = {0.f, 0.f, 0.f, 0.f};
  if (on) {
    f32x4 w[4] = {};
    int u = wave;
    for (; u + 12 < n; u += 16)
#pragma unroll
      for (int q = 0; q < 4; ++q) w[q] += *reinterpret_cast<const f32x4*>(p + (u + 4 * q) * step);
    for (; u < n; u += 4) w[0] += *reinterpret_cast<const f32x4*>(p + u * step);
    v = (w[0] + w[1]) + (w[2] + w[3]);
  }
  quarter[wave][lane] = v;
  __syncthreads();
  if (wave == 0 && on) {
    v = (quarter[0][lane] + quarter[1][lane]) + (quarter[2][lane] + quarter[3][lane]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      if (bias) {
        if (i - size + q < N) db[(int64_t)e * N + (i - size) + q] = from_f32<T>(v[q]);
      } else {
        const int64_t m = (i + q) / ldo, c = (i + q) % ldo;
        if (c < K) dw[((int64_t)e * N + m) * K + c] = from_f32<T>(v[q]);
      }
    }
  }
}

// ... of every expert
template <typename T>
__global__ __launch_bounds__(256) void dw_join_kernel(const float* __restrict__ parts, const float* __restrict__ db_parts, const int* __restrict__ offsets,
                                                      int64_t M, int N, int K, int ldo, int piece, T* __restrict__ dw, T* __restrict__ db) {
  __shared__ int wave_sum[4];
  const int e = blockIdx.y;
  int before = 0;
  for (int i = threadIdx.x; i < e; i += 256) {
    const int64_t lo = bounded(offsets[i], M), hi = bounded(offsets[i + 1], M);
    if (hi > lo) before += (int)((hi - lo + piece - 1) / piece);
  }
  for (int d = 32; d > 0; d >>= 1) before += __shfl_xor(before, d, 64);
  if ((threadIdx.x & 63) == 0) wave_sum[threadIdx.x >> 6] = before;
  __syncthreads();
  const int64_t most = row_tiles_at_most(M, gridDim.y, piece), all = (int64_t)wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
  const int64_t first = all < most ? all : most, lo = bounded(offsets[e], M), hi = bounded(offsets[e + 1], M);
  const int64_t mine = hi > lo ? (hi - lo + piece - 1) / piece : 0;
  join_pieces(parts, db_parts, e, first, (int)(mine < most - first ? mine : most - first), blockIdx.x, N, K, ldo, dw, db);
}

// ... of the experts with more than `piece` rows: the workgroups of a row of the grid look at every gridDim.y-th piece, and where it is its
// expert's first share out the sums
template <typename T>
__global__ __launch_bounds__(256) void dw_join_crowded_kernel(const float* __restrict__ parts, const float* __restrict__ db_parts,
                                                              const int* __restrict__ offsets, int64_t M, int E, int N, int K, int ldo, int piece, int chunks,
                                                              T* __restrict__ dw, T* __restrict__ db) {
  const RowTiles pieces(offsets, E, M, piece, piece);
  for (int u = blockIdx.y; u < pieces.total; u += gridDim.y) {
    const RowTile t = pieces.find(u);
    const int64_t lo = bounded(offsets[t.expert], M), n = (bounded(offsets[t.expert + 1], M) - lo + piece - 1) / piece;
    if (t.row0 != lo) continue;
    for (int chunk = blockIdx.x; chunk < chunks; chunk += gridDim.x) {
      join_pieces(parts, db_parts, t.expert, u, (int)(n < pieces.total - u ? n : pieces.total - u), chunk, N, K, ldo, dw, db);
      __syncthreads();
    }
  }
}

// rows of `cols` elements `ld` apart -> rows of whole 16-byte chunks, zeros behind the last element (5003 x 385 fp16: 4 us); two operands at once
template <typename T>
struct PackJob {
  const T* src;
  int64_t ld, chunks;  // chunks: of all rows
  int cols, across;    // across: chunks of a row
  T* dst;
};
template <typename T>
__global__ __launch_bounds__(256) void pack_rows_kernel(PackJob<T> a, PackJob<T> b) {
  for (int64_t id = (int64_t)blockIdx.x * 256 + threadIdx.x; id < a.chunks + b.chunks; id += (int64_t)gridDim.x * 256) {
    const PackJob<T>& job = id < a.chunks ? a : b;
    const int64_t at = id < a.chunks ? id : id - a.chunks, row = at / job.across;
    const int c = (int)(at % job.across) * kChunk<T>;
    const T* src = job.src + row * job.ld + c;
    Pack<T, kChunk<T>> o;
    if (c + kChunk<T> <= job.cols) {
      o = load_any<T, kChunk<T>>(src);
    } else {
#pragma unroll
      for (int q = 0; q < kChunk<T>; ++q) o.v[q] = c + q < job.cols ? src[q] : from_f32<T>(0.0f);
    }
    store_pack(job.dst + at * kChunk<T>, o);
  }
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == kF32) return f(float{});
  if (dtype == kF16) return f(_Float16{});
  if (dtype == kBF16) return f(__bf16{});
  ps_set_error("unknown element type (0 fp32, 1 fp16, 2 bf16)");
  return -1;
}

constexpr int64_t kMaxWidth = 1 << 20;

bool sizes_ok(int64_t M, int E, int64_t n_in, int64_t n_out) {
  return M >= 0 && M < ((int64_t)1 << 31) - (1 << 20) && E >= 1 && E <= 65536 && n_in >= 1 && n_in <= kMaxWidth && n_out >= 1 && n_out <= kMaxWidth;
}

constexpr int kCompute = 256;  // compute units

// What a step of k (128 bytes of it) of a 64, 128 or 256 tile was measured to take, us: of its compute unit's time (the reads from the L2; in fp32
// the matrix instructions, of which 256 would spare none), and at least from its start to its end
struct StepCost {
  int sizes;
  double busy[3], least[3];
};
StepCost step_cost(int dtype) {
  if (dtype == kF32) return {2, {0.47, 1.75}, {0.8, 1.75}};
  return {3, {0.27, 0.73, 2.1}, {0.45, 0.8, 2.1}};
}

// Tile sizes: the cheapest by these, of those that an expert's share of the rows fills for the most part (bf16: 65536 rows, 32 experts of 2048 x
// 1024 with 256 316 us, with 128 375; 16384, 8 of 1024 x 1024 35 and 42; 128 rows each, 64 experts of 1024 x 1024 with 128 28 us, with 64 32; 64
// rows each, 512 x 512 11.2 and 9.4; fp32, 740 rows, 3 of 495 -> 80 with 128 45, with 64 20).
// Few tiles and a long k: k is shared out over as many workgroups per tile as two per compute unit allow, of at least four steps, where that
// saves more than 7 us, the second launch's and its way through the memory (1 row, 2048 -> 2048 bf16 13.0 -> 8.1 us, 4096 -> 64 fp32 87 -> 10).
struct LinearPlan {
  int tile, parts;
};
LinearPlan linear_plan(int64_t rows, int64_t groups, int64_t cols, int64_t k, int dtype) {
  const StepCost cost = step_cost(dtype);
  const int64_t each = rows / groups;
  LinearPlan best{64, 1};
  double best_us = 1e30;
  for (int i = 0; i < cost.sizes; ++i) {
    const int tile = 64 << i;
    if (i > 0 && (cols <= tile / 2 || each * 4 < tile * 3)) break;
    const double shared = ((double)rows / tile + 0.5 * groups) * (double)((cols + tile - 1) / tile) / kCompute;  // tiles per compute unit
    const double us = cost.busy[i] * shared > cost.least[i] ? cost.busy[i] * shared : cost.least[i];
    if (us <= best_us) best.tile = tile, best_us = us;
  }
  if (best.tile == 64) {
    const int step = dtype == kF32 ? 32 : 64;
    const int64_t tiles = row_tiles_at_most(rows, (int)groups, 64) * ((cols + 63) / 64), steps = (k + step - 1) / step;
    const int64_t room = tiles > 0 ? 2 * kCompute / tiles : 0, parts = room < steps / 4 ? room : steps / 4;
    if (parts > 1 && (double)(steps - steps / parts) * cost.least[0] > 7.0) best.parts = (int)parts;
  }
  return best;
}
int64_t share_bytes(const LinearPlan& p, int64_t rows, int64_t cols) { return p.parts > 1 ? (p.parts * rows * cols * 4 + 255) & ~(int64_t)255 : 0; }

template <typename K>
void allow_lds(K* kernel, int bytes) {
  if (bytes > 64 * 1024) hipFuncSetAttribute((const void*)kernel, hipFuncAttributeMaxDynamicSharedMemorySize, bytes);
}

// An operand as the products read it: rows of whole 16-byte chunks that start on 16 bytes
struct Rows {
  const void* p;
  int64_t ld;
};
int size_of(int dtype) { return dtype == kF32 ? 4 : 2; }
int64_t padded(int64_t cols, int dtype) {
  const int chunk = 16 / size_of(dtype);
  return (cols + chunk - 1) / chunk * chunk;
}
bool is_packed(const void* p, int64_t ld, int64_t cols, int dtype) {
  const int size = size_of(dtype);
  return ((uintptr_t)p & 15) == 0 && ((ld * size) & 15) == 0 && ((cols * size) & 15) == 0;
}
int64_t pack_bytes(const void* p, int64_t ld, int64_t rows, int64_t cols, int dtype) {
  return is_packed(p, ld, cols, dtype) ? 0 : (rows * padded(cols, dtype) * size_of(dtype) + 255) & ~(int64_t)255;
}
// two operands as they are, or their copies from `to` on
struct Operand {
  const void* p;
  int64_t ld, rows, cols;
};
template <typename T>
void packed(const Operand& a, const Operand& b, int dtype, char* to, Rows* as, Rows* bs, hipStream_t s) {
  auto job = [&](const Operand& o, Rows* r) {
    const int64_t bytes = pack_bytes(o.p, o.ld, o.rows, o.cols, dtype);
    const int across = (int)(padded(o.cols, dtype) / kChunk<T>);
    PackJob<T> j{(const T*)o.p, o.ld, bytes == 0 ? 0 : o.rows * across, (int)o.cols, across, (T*)to};
    *r = bytes == 0 ? Rows{o.p, o.ld} : Rows{to, padded(o.cols, dtype)};
    to += bytes;
    return j;
  };
  const PackJob<T> ja = job(a, as), jb = job(b, bs);
  if (ja.chunks + jb.chunks > 0) pack_rows_kernel<T><<<blocks_of_256(ja.chunks + jb.chunks), 256, 0, s>>>(ja, jb);
}

template <typename T, int B, int WM, int WN, bool W_RC, bool SHARED>
int launch_linear_tile(const Rows& x, const Rows& w, int w_rows, const void* bias, const int32_t* offsets, int64_t M, int E, int N, int K, int parts, void* y,
                       hipStream_t s) {
  constexpr int lds = 4 * B * kTileRowBytes;
  const int64_t blocks = xcd_blocks(row_tiles_at_most(M, E, B) * ((N + B - 1) / B) * parts + 1);
  PS_REQUIRE(blocks * 64 * WM * WN < kMaxThreads, "ps_expert_linear: too many tiles");
  allow_lds(linear_kernel<T, B, B, WM, WN, W_RC, SHARED>, lds);
  linear_kernel<T, B, B, WM, WN, W_RC, SHARED><<<(unsigned)blocks, 64 * WM * WN, lds, s>>>(
      (const T*)x.p, x.ld, (const T*)w.p, w.ld, w_rows, (const T*)bias, offsets, M, E, N, K, parts, (std::conditional_t<SHARED, float, T>*)y);
  PS_CHECK_LAUNCH();
}

// x [M,K] (dy) times the weights [E,out,in]: W_RC = false: K = in, N = out; true: K = out, N = in
template <bool W_RC>
int launch_linear(const void* x, int64_t ldx, const void* weight, const void* bias, const int32_t* offsets, int64_t M, int E, int64_t n_in, int64_t n_out,
                  int dtype, void* y, void* workspace, hipStream_t s) {
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int64_t k = W_RC ? n_out : n_in;
    const int N = (int)(W_RC ? n_in : n_out), K = (int)padded(k, dtype), rows = (int)n_out;
    const LinearPlan p = linear_plan(M, E, N, k, dtype);
    Rows xs, ws;
    packed<T>({x, ldx, M, k}, {weight, n_in, E * n_out, n_in}, dtype, (char*)workspace + share_bytes(p, M, N), &xs, &ws, s);
    if (p.parts > 1) {
      const int rc = launch_linear_tile<T, 64, 2, 2, W_RC, true>(xs, ws, rows, bias, offsets, M, E, N, K, p.parts, workspace, s);
      if (rc != 0) return rc;
      linear_join_kernel<T><<<(unsigned)((M * N + 255) / 256), 256, 0, s>>>((const float*)workspace, p.parts, offsets, E, M, N, (T*)y);
      PS_CHECK_LAUNCH();
    }
    if constexpr (sizeof(T) == 2)
      if (p.tile == 256) return launch_linear_tile<T, 256, 2, 4, W_RC, false>(xs, ws, rows, bias, offsets, M, E, N, K, 1, y, s);
    if (p.tile == 128) return launch_linear_tile<T, 128, 2, 2, W_RC, false>(xs, ws, rows, bias, offsets, M, E, N, K, 1, y, s);
    return launch_linear_tile<T, 64, 2, 2, W_RC, false>(xs, ws, rows, bias, offsets, M, E, N, K, 1, y, s);
  });
}

// How the weight gradients are cut: the tile, the rows of a piece and the pieces that there are room for
struct DwPlan {
  DwCut cut;
  int tile, piece;
  int64_t units;
};
// The cheapest by the tiles' steps.  Pieces shorten the longest run of steps and cost 5 us and the way of their fp32 sums through the memory,
// 4.5 TB/s; without them an expert may well have twice its share of the rows.  Where one that had them all would keep its compute units busy for
// more than 150 us (a router that has collapsed), those with more than four times their share, 2048 rows, and what it takes of all rows for two
// workgroups per compute unit, are cut all the same: a launch more, which finds nothing to join as a rule, and room for half as many sums as there
// are experts, or as 1024 tiles hold, at most.  No sum is then longer than that, and no longer than 150 us of steps otherwise.
//     evenly shared / all rows to one expert, cut and not:  131072 rows, 1024 experts of 64 x 64 fp32 24 / 75 us, 20 / 4090 | 65536, 128 of 256 x 256
//     fp32 92 / 191, 84 / 5566 | 65536, 32 of 2048 x 1024 bf16 277 / 298, 275 / 1769 | 16384, 8 of 1024 x 1024 bf16 43 / 107, 43 / 225
//     16 experts, fp32:  131072 rows of 64 x 64 in pieces 22 us, whole 191 | 32768 rows of 128 x 128 in pieces, tiles of 64 21, of 128 30
//     bf16:  8192 rows, 16 experts of 512 x 512 whole 12, in pieces 45 | 65536 rows, 32 experts of 2048 x 1024 tiles of 256 307, of 128 374
DwPlan dw_plan(int64_t M, int E, int64_t n_in, int64_t n_out, int dtype) {
  const bool wide = dtype == kF32;
  const StepCost cost = step_cost(dtype);
  const int64_t least = n_in < n_out ? n_in : n_out, step_rows = wide ? 32 : 64, each = M / E;
  DwPlan best{kWhole, 64, 0, 0};
  double best_us = 1e30;
  for (int i = 0; i < cost.sizes; ++i) {
    const int tile = 64 << i;
    if (i > 0 && least <= tile / 2) break;
    const double tiles = (double)((n_in + tile - 1) / tile) * ((n_out + tile - 1) / tile);
    for (int64_t pieces = 1; pieces == 1 || each / pieces >= 192; pieces *= 2) {
      DwPlan p{kWhole, tile, 0, 0};
      int64_t rows = each, longest = E > 1 ? 2 * each : each;
      double more = 0.0;  // what the pieces cost
      if (pieces > 1) {
        rows = ((each + pieces - 1) / pieces + 63) & ~(int64_t)63;
        longest = rows = rows < 256 ? 256 : rows;
        p = {kPieces, tile, (int)rows, row_tiles_at_most(M, E, (int)rows)};
        more = 5.0 + 8e-6 / 4.5 * p.units * n_in * n_out;
      } else if (cost.least[i] * (double)((M + step_rows - 1) / step_rows) > 150.0) {
        const double share = 4.0 * (double)M / E, full = (double)M * tiles / (2 * kCompute);
        const int64_t most = ((int64_t)(share > full ? (share > 2048 ? share : 2048) : (full > 2048 ? full : 2048)) + 63) & ~(int64_t)63;
        if (most < M) p = {kCrowded, tile, (int)most, crowded_pieces_at_most(M, (int)most)}, more = 3.0;
      }
      const double shared = tiles * (pieces > 1 ? (double)M / rows + 0.5 * E : (double)E) / kCompute;  // workgroups per compute unit
      const double steps = (double)((rows + step_rows - 1) / step_rows), all = cost.busy[i] * (shared > 1 ? shared : 1) * (steps > 1 ? steps : 1);
      const double run = cost.least[i] * (double)((longest + step_rows - 1) / step_rows);
      const double us = (all > run ? all : run) + more;
      if (us < best_us) best = p, best_us = us;
    }
  }
  return best;
}

int64_t round4(int64_t v) { return (v + 3) / 4 * 4; }
int64_t dw_part_bytes(const DwPlan& p, int64_t n_in, int64_t n_out) {
  return p.cut == kWhole ? 0 : (p.units * (n_out * round4(n_in) + round4(n_out)) * (int64_t)sizeof(float) + 255) & ~(int64_t)255;
}

struct DwArgs {
  const int32_t* offsets;
  int64_t M;
  int E, N, K, ldo;
  void *dw, *db;
  float *parts, *db_parts;
};
template <typename T, int B, int WM, int WN, DwCut CUT>
int launch_dw_tile(const DwPlan& p, const Rows& dy, const Rows& x, const DwArgs& d, hipStream_t s) {
  constexpr int lds = 4 * B * kTileRowBytes;
  const int64_t tiles = ((d.N + B - 1) / B) * (int64_t)((d.K + B - 1) / B), pieces = CUT == kWhole ? 0 : xcd_blocks(p.units * tiles);
  const int64_t blocks = pieces + (CUT == kPieces ? 0 : xcd_blocks(d.E * tiles));
  PS_REQUIRE(blocks * 64 * WM * WN < kMaxThreads, "ps_expert_linear_dw: too many tiles");
  allow_lds(linear_dw_kernel<T, B, B, WM, WN, CUT>, lds);
  linear_dw_kernel<T, B, B, WM, WN, CUT><<<(unsigned)blocks, 64 * WM * WN, lds, s>>>((const T*)dy.p, dy.ld, (const T*)x.p, x.ld, d.offsets, d.M, d.E, d.N, d.K,
                                                                                    d.ldo, p.piece, (int)pieces, d.dw, d.db, d.parts, d.db_parts);
  PS_CHECK_LAUNCH();
}

template <typename T, DwCut CUT>
int launch_dw(const DwPlan& p, const Rows& dy, const Rows& x, const DwArgs& d, hipStream_t s) {
  if constexpr (sizeof(T) == 2)
    if (p.tile == 256) return launch_dw_tile<T, 256, 2, 4, CUT>(p, dy, x, d, s);
  if (p.tile == 128) return launch_dw_tile<T, 128, 2, 2, CUT>(p, dy, x, d, s);
  return launch_dw_tile<T, 64, 2, 2, CUT>(p, dy, x, d, s);
}

enum Pass { kForward, kInputGradient, kWeightGradient };

int64_t workspace_of(int pass, const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t M, int E, int64_t n_in, int64_t n_out, int dtype) {
  if (pass == kWeightGradient)
    return dw_part_bytes(dw_plan(M, E, n_in, n_out, dtype), n_in, n_out) + pack_bytes(a, a_stride, M, n_out, dtype) + pack_bytes(b, b_stride, M, n_in, dtype);
  const int64_t k = pass == kForward ? n_in : n_out, n = pass == kForward ? n_out : n_in;
  return share_bytes(linear_plan(M, E, n, k, dtype), M, n) + pack_bytes(a, a_stride, M, k, dtype) + pack_bytes(b, n_in, E * n_out, n_in, dtype);
}

}  // namespace

extern "C" int64_t ps_expert_linear_workspace(int pass, const void* a, int64_t a_stride, const void* b, int64_t b_stride, int64_t M, int E, int64_t n_in,
                                              int64_t n_out, int dtype) {
  if (!sizes_ok(M, E, n_in, n_out) || pass < kForward || pass > kWeightGradient || dtype < kF32 || dtype > kBF16) return 0;
  return workspace_of(pass, a, a_stride, b, b_stride, M, E, n_in, n_out, dtype);
}

extern "C" int ps_expert_linear_fwd(const void* x, int64_t x_stride, const void* weight, const void* bias, const int32_t* offsets, int64_t M, int E,
                                    int64_t n_in, int64_t n_out, int dtype, void* y, void* workspace, void* stream) {
  PS_REQUIRE(sizes_ok(M, E, n_in, n_out) && x_stride >= n_in && x_stride <= kMaxWidth, "ps_expert_linear_fwd: sizes out of range");
  if (M == 0) return 0;
  PS_REQUIRE(x != nullptr && weight != nullptr && offsets != nullptr && y != nullptr, "ps_expert_linear_fwd: null argument");
  PS_REQUIRE(workspace != nullptr || workspace_of(kForward, x, x_stride, weight, n_in, M, E, n_in, n_out, dtype) == 0,
             "ps_expert_linear_fwd: needs its workspace (ps_expert_linear_workspace)");
  return launch_linear<false>(x, x_stride, weight, bias, offsets, M, E, n_in, n_out, dtype, y, workspace, (hipStream_t)stream);
}

extern "C" int ps_expert_linear_dx(const void* dy, int64_t dy_stride, const void* weight, const int32_t* offsets, int64_t M, int E, int64_t n_in,
                                   int64_t n_out, int dtype, void* dx, void* workspace, void* stream) {
  PS_REQUIRE(sizes_ok(M, E, n_in, n_out) && dy_stride >= n_out && dy_stride <= kMaxWidth, "ps_expert_linear_dx: sizes out of range");
  if (M == 0) return 0;
  PS_REQUIRE(dy != nullptr && weight != nullptr && offsets != nullptr && dx != nullptr, "ps_expert_linear_dx: null argument");
  PS_REQUIRE(workspace != nullptr || workspace_of(kInputGradient, dy, dy_stride, weight, n_in, M, E, n_in, n_out, dtype) == 0,
             "ps_expert_linear_dx: needs its workspace (ps_expert_linear_workspace)");
  return launch_linear<true>(dy, dy_stride, weight, nullptr, offsets, M, E, n_in, n_out, dtype, dx, workspace, (hipStream_t)stream);
}

extern "C" int ps_expert_linear_dw(const void* dy, int64_t dy_stride, const void* x, int64_t x_stride, const int32_t* offsets, int64_t M, int E,
                                   int64_t n_in, int64_t n_out, int dtype, void* dweight, void* dbias, void* workspace, void* stream) {
  PS_REQUIRE(sizes_ok(M, E, n_in, n_out) && x_stride >= n_in && x_stride <= kMaxWidth && dy_stride >= n_out && dy_stride <= kMaxWidth,
             "ps_expert_linear_dw: sizes out of range");
  PS_REQUIRE((M == 0 || (dy != nullptr && x != nullptr)) && offsets != nullptr && dweight != nullptr, "ps_expert_linear_dw: null argument");
  PS_REQUIRE(workspace != nullptr || workspace_of(kWeightGradient, dy, dy_stride, x, x_stride, M, E, n_in, n_out, dtype) == 0,
             "ps_expert_linear_dw: needs its workspace (ps_expert_linear_workspace)");
  const DwPlan p = dw_plan(M, E, n_in, n_out, dtype);
  const int N = (int)n_out, K = (int)n_in, ldo = (int)round4(n_in);
  hipStream_t s = (hipStream_t)stream;
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    float* parts = (float*)workspace;
    Rows dys, xs;
    packed<T>({dy, dy_stride, M, n_out}, {x, x_stride, M, n_in}, dtype, (char*)workspace + dw_part_bytes(p, n_in, n_out), &dys, &xs, s);
    float* db_parts = parts + p.units * n_out * ldo;
    const DwArgs d{offsets, M, E, N, K, ldo, dweight, dbias, parts, db_parts};
    if (p.cut == kWhole) return launch_dw<T, kWhole>(p, dys, xs, d, s);
    const int rc = p.cut == kPieces ? launch_dw<T, kPieces>(p, dys, xs, d, s) : launch_dw<T, kCrowded>(p, dys, xs, d, s);
    if (rc != 0) return rc;
    const int64_t sums = n_out * ldo + (dbias != nullptr ? round4(n_out) : 0);
    const unsigned chunks = (unsigned)((sums + 255) / 256);
    if (p.cut == kPieces)
      dw_join_kernel<T><<<dim3(chunks, (unsigned)E), 256, 0, s>>>(parts, db_parts, offsets, M, N, K, ldo, p.piece, (T*)dweight, (T*)dbias);
    else {  // (as a rule there is nothing to do: few workgroups)
      const unsigned across = chunks < 512 ? chunks : 512, most = across < 256 ? 256 / across : 1;
      dw_join_crowded_kernel<T><<<dim3(across, p.units < most ? (unsigned)p.units : most), 256, 0, s>>>(parts, db_parts, offsets, M, E, N, K, ldo, p.piece,
                                                                                                       (int)chunks, (T*)dweight, (T*)dbias);
    }
    PS_CHECK_LAUNCH();
  });
}
