// The orthogonalised update: a batch of matrices G [B, m, n], each scaled to Frobenius norm one and pushed `steps` times through the odd
// polynomial  X <- a X + (b S + c S^2) X,  S = X X^T,  that moves singular values towards one (Newton-Schulz).  X is kept short side
// first: [s, l] with s = min(m, n), l = max(m, n), so both products of a step with X and the square of S have the fewest operations.
//
// Arithmetic.  The polynomial multiplies what rounding leaves in the small singular directions by up to a^steps, so one 16-bit rounding
// per step is not enough for an fp32 result.  Every matrix is kept as a PAIR of fp16 planes, value = (hi + lo) / 1024: 22 bits and the
// sign, and a product is three matrix instructions, hi hi + hi lo + lo hi, summed in fp32 (lo lo, 2^-24 of the product, is left out).
// That is fp32's own precision at a third of the fp16 rate, five times the fp32 matrix rate.
//
// Range.  The planes hold X^ = X / r with r = norm / (norm + eps) at the start, so an input far below eps loses nothing; a step
// multiplies r by the power of two `grow` that bounds a + b t + c t^2, until r passes 1/2, and keeps it from then on.  The caller
// checks that the iterates' squared singular values and the polynomial stay under 15: with X^ <= 2 X all entries are below 64, the
// planes' end, and 1024 * entry keeps the low half normal down to entries of 2^-12.
#include "gemm_core.hpp"

namespace {

using namespace ps;

constexpr float kPlaneScale = 1024.0f;                       // fp16 planes hold 1024 * value
constexpr float kProductScale = 1.0f / (1024.0f * 1024.0f);  // of a product of two
constexpr int kNormParts = 64;                               // partial sums of squares per matrix

template <typename V>  // float or double
__device__ __forceinline__ void split(V v, _Float16& hi, _Float16& lo) {
  const V t = v * (V)kPlaneScale;
  hi = (_Float16)(float)t;
  lo = (_Float16)(float)(t - (V)(float)hi);
}

struct Shape {  // of one matrix
  int64_t m, n;      // as given
  int s, l;          // short and long side
  int sp, lp;        // rounded up to whole tiles of k (zeros there)
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

// Workspace of a batch: pairs of planes (hi, then lo, for all matrices)
struct Work {
  _Float16 *x, *xt[2], *gram, *poly;  // [B][s][lp], [B][l][sp] twice, [B][s][sp], [B][s][sp]
  double* norms;                      // [B][kNormParts]
  float* ratio;                       // [B] r at the start
  int64_t x_plane, xt_plane, s_plane, bytes;
};
Work work_of(const Shape& h, int64_t B, void* base) {
  Work w;
  w.x_plane = B * h.s * (int64_t)h.lp;
  w.xt_plane = B * h.l * (int64_t)h.sp;
  w.s_plane = B * h.s * (int64_t)h.sp;
  char* p = (char*)base;
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) & ~(int64_t)255;
    return q;
  };
  w.norms = (double*)take(B * kNormParts * 8);
  w.ratio = (float*)take(B * 4);
  w.x = (_Float16*)take(w.x_plane * 4);
  w.xt[0] = (_Float16*)take(w.xt_plane * 4);
  w.xt[1] = (_Float16*)take(w.xt_plane * 4);
  w.gram = (_Float16*)take(w.s_plane * 4);
  w.poly = (_Float16*)take(w.s_plane * 4);
  w.bytes = p - (char*)base;
  return w;
}

// Where the matrix comes from: G itself, or an optimizer's momentum buf <- mu buf + (1 - mu) g, taken as it is or (nesterov) as
// mu buf + (1 - mu) g once more
struct Source {
  const void* g;
  float* buf;  // null: g alone
  float mu, nu;  // momentum, 1 - momentum
  int nesterov;
};

template <typename T, bool MOMENTUM, bool UPDATE>
__device__ __forceinline__ float source_value(const Source& src, int64_t i) {
#pragma clang fp contract(off)  // the same bits in both passes over the source
  const float g = to_f32(reinterpret_cast<const T*>(src.g)[i]);
  if constexpr (!MOMENTUM) return g;
  float b = src.buf[i];
  if constexpr (UPDATE) {
    b = src.mu * b + src.nu * g;
    src.buf[i] = b;
  }
  return src.nesterov ? src.mu * b + src.nu * g : b;
}

// partial sums of squares, in 64 bits: entries of any fp32 size neither overflow nor vanish
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_norm_kernel(Source src, int64_t size, double* __restrict__ norms) {
  __shared__ double part[4];
  const int64_t base = (int64_t)blockIdx.y * size;
  double sum = 0.0;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < size; i += kNormParts * 256) {
    const double v = source_value<T, MOMENTUM, true>(src, base + i);
    sum += v * v;
  }
  for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, 64);
  if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = sum;
  __syncthreads();
  if (threadIdx.x == 0) norms[(int64_t)blockIdx.y * kNormParts + blockIdx.x] = (part[0] + part[1]) + (part[2] + part[3]);
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

// X^ = G / norm as planes, both ways round, 32 x 32 elements at a time; zeros in the padding of either
template <typename T, bool MOMENTUM>
__global__ __launch_bounds__(256) void ns_start_kernel(Source src, Shape h, Work w, float eps) {
  __shared__ double tile[32][33];
  __shared__ double inv;
  const int64_t b = blockIdx.z;
  if (threadIdx.x == 0) {
    double sum = 0.0;
    for (int i = 0; i < kNormParts; ++i) sum += w.norms[b * kNormParts + i];
    const double norm = sqrt(sum);
    inv = norm == 0.0 ? 0.0 : 1.0 / norm;
    if (blockIdx.x == 0 && blockIdx.y == 0) w.ratio[b] = norm == 0.0 ? 0.0f : (float)(norm / (norm + (double)eps));
  }
  __syncthreads();
  const int rows = h.tall ? h.l : h.s, cols = h.tall ? h.s : h.l;  // as given: [m, n]
  const int r0 = blockIdx.y * 32, c0 = blockIdx.x * 32, tx = threadIdx.x & 31, ty = threadIdx.x >> 5;
  const int64_t base = b * h.m * h.n;
  for (int k = ty; k < 32; k += 8) {
    const int r = r0 + k, c = c0 + tx;
    tile[k][tx] = r < rows && c < cols ? source_value<T, MOMENTUM, false>(src, base + (int64_t)r * h.n + c) * inv : 0.0;
  }
  __syncthreads();
  // plane rows along the given rows, and along the given columns
  _Float16* same = h.tall ? w.xt[0] : w.x;
  _Float16* turned = h.tall ? w.x : w.xt[0];
  const int64_t same_plane = h.tall ? w.xt_plane : w.x_plane, turned_plane = h.tall ? w.x_plane : w.xt_plane;
  const int same_ld = h.tall ? h.sp : h.lp, turned_ld = h.tall ? h.lp : h.sp;
  for (int k = ty; k < 32; k += 8) {
    _Float16 hi, lo;
    if (r0 + k < rows && c0 + tx < same_ld) {
      split(tile[k][tx], hi, lo);
      const int64_t at = (b * rows + r0 + k) * same_ld + c0 + tx;
      same[at] = hi;
      same[same_plane + at] = lo;
    }
    if (c0 + k < cols && r0 + tx < turned_ld) {
      split(tile[tx][k], hi, lo);
      const int64_t at = (b * cols + c0 + k) * turned_ld + r0 + tx;
      turned[at] = hi;
      turned[turned_plane + at] = lo;
    }
  }
}

// ------------------------------------------------------------------------------------------------ products of pairs
enum Product {
  kGram,   // S = X X^T                            rows of X     x rows of X,    k = l
  kPoly,   // P = a I + b S + c S S                rows of S     x rows of S,    k = s    (S is symmetric)
  kApply,  // X' = P X, both ways round            rows of P     x rows of X^T,  k = s
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

struct Operands {
  const _Float16 *a, *b;      // [B][ra][k], [B][rb][k]; the lo plane is a_plane / b_plane behind
  int64_t a_plane, b_plane;
  int ra, rb, k;              // k: padded, and the rows' distance
};

constexpr int kPairTile = 128;

template <typename T, Product WHAT>
__global__ __launch_bounds__(256) void ns_product_kernel(Operands o, Shape h, Work w, int step, Poly c, Result res) {
  constexpr int BM = kPairTile, BN = kPairTile, NT = 256, MI = 4, NJ = 4;
  constexpr int kPart = BM * kTileRowBytes;  // bytes of one plane's tile
  __shared__ __attribute__((aligned(16))) char lds[4 * kPart];
  const int tm_n = (o.ra + BM - 1) / BM, tn_n = (o.rb + BN - 1) / BN;
  const int tn = blockIdx.x % tn_n, tm = blockIdx.x / tn_n % tm_n;
  const int64_t batch = blockIdx.x / (tn_n * tm_n);
  const int m0 = tm * BM, n0 = tn * BN;
  const int rows = o.ra - m0 < BM ? o.ra - m0 : BM, cols = o.rb - n0 < BN ? o.rb - n0 : BN;
  const _Float16* a = o.a + (batch * o.ra + m0) * o.k;
  const _Float16* b = o.b + (batch * o.rb + n0) * o.k;
  const unsigned ld = (unsigned)o.k * 2;
  TileLoader<_Float16, BM, NT, 16, false> ah, al, bh, bl;
  auto load = [&](int k0) {
    const int64_t abytes = ((int64_t)(rows - 1) * o.k + (o.k - k0)) * 2, bbytes = ((int64_t)(cols - 1) * o.k + (o.k - k0)) * 2;
    ah.load(window(a + k0, abytes), ld, o.k - k0);
    al.load(window(a + o.a_plane + k0, abytes), ld, o.k - k0);
    bh.load(window(b + k0, bbytes), ld, o.k - k0);
    bl.load(window(b + o.b_plane + k0, bbytes), ld, o.k - k0);
  };
  // the two small products add up apart from the large one: each of their additions to it would cost it another rounding
  f32x4 acc[MI][NJ], fine[MI][NJ];
#pragma unroll
  for (int i = 0; i < MI; ++i)
#pragma unroll
    for (int j = 0; j < NJ; ++j) acc[i][j] = fine[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  const int wave = threadIdx.x >> 6, wm = (wave >> 1) * 64, wn = (wave & 1) * 64;
  load(0);
  for (int k0 = 0; k0 < o.k; k0 += 64) {
    __syncthreads();
    ah.store(lds);
    al.store(lds + kPart);
    bh.store(lds + 2 * kPart);
    bl.store(lds + 3 * kPart);
    __syncthreads();
    if (k0 + 64 < o.k) load(k0 + 64);
    tile_mma<_Float16, MI, NJ>(lds, lds + 2 * kPart, wm, wn, acc);
    tile_mma<_Float16, MI, NJ>(lds, lds + 3 * kPart, wm, wn, fine);
    tile_mma<_Float16, MI, NJ>(lds + kPart, lds + 2 * kPart, wm, wn, fine);
  }
  const float ratio = ratio_at(w.ratio[batch], step, c.grow);
  // kPoly: a + b r^2 S^ + c r^4 S^ S^, formed in 64 bits: an error of a coefficient would be common to all entries and grow like a
  // singular value's, and it is the small product of a step | kApply: over the step's growth of r | kLast: X = r X^
  const double r2 = (double)ratio * ratio, pb = c.b * r2 / kPlaneScale, pc = c.c * r2 * r2 * kProductScale;
  const float out_scale = WHAT == kApply ? kProductScale * (ratio > 0.0f ? ratio / ratio_at(ratio, 1, c.grow) : 1.0f)
                                         : (WHAT == kLast ? kProductScale * ratio : kProductScale);
  _Float16* const xt_next = w.xt[(step + 1) & 1];
  const int r = threadIdx.x & 15, g = (threadIdx.x >> 4) & 3;
#pragma unroll
  for (int i = 0; i < MI; ++i) {
    const int m = m0 + wm + i * 16 + r;
    if (m >= (WHAT == kApply ? h.sp : o.ra)) continue;
#pragma unroll
    for (int j = 0; j < NJ; ++j)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int n = n0 + wn + j * 16 + g * 4 + q;
        const float sum = acc[i][j][q] + fine[i][j][q];
        float v = sum * out_scale;
        _Float16 hi, lo;
        if constexpr (WHAT == kGram || WHAT == kPoly) {
          if (n >= h.sp) continue;
          const int64_t at = (batch * h.s + m) * h.sp + n;
          if (n >= h.s) {
            hi = lo = (_Float16)0.0f;  // the padding of k in the products to come
          } else if constexpr (WHAT == kPoly) {
            split(pc * sum + (pb * ((double)(float)w.gram[at] + (double)(float)w.gram[w.s_plane + at]) + (m == n ? c.a : 0.0)), hi, lo);
          } else {
            split(v, hi, lo);
          }
          _Float16* out = WHAT == kGram ? w.gram : w.poly;
          out[at] = hi;
          out[w.s_plane + at] = lo;
        } else if constexpr (WHAT == kApply) {
          if (n >= h.lp) continue;
          if (n >= h.l || m >= h.s) v = 0.0f;  // the padding of k, both ways round
          split(v, hi, lo);
          if (m < h.s) {
            const int64_t at = (batch * h.s + m) * h.lp + n;
            w.x[at] = hi;
            w.x[w.x_plane + at] = lo;
          }
          if (n < h.l) {
            const int64_t t = (batch * h.l + n) * h.sp + m;
            xt_next[t] = hi;
            xt_next[w.xt_plane + t] = lo;
          }
        } else {
          if (n >= h.l) continue;
          const int64_t at = batch * h.m * h.n + (h.tall ? (int64_t)n * h.n + m : (int64_t)m * h.n + n);
          if (res.update) {
            float* p = reinterpret_cast<float*>(res.out) + at;
            *p = res.keep * *p - res.rate * v;
          } else {
            reinterpret_cast<T*>(res.out)[at] = from_f32<T>(v);
          }
        }
      }
  }
}

int64_t pair_tiles(int64_t ra, int64_t rb, int64_t B) { return ((ra + kPairTile - 1) / kPairTile) * ((rb + kPairTile - 1) / kPairTile) * B; }

template <typename T, Product WHAT>
void launch_product(const Operands& o, const Shape& h, const Work& w, int64_t B, int step, const Poly& c, const Result& res, hipStream_t s) {
  const int64_t tiles = pair_tiles(o.ra, o.rb, B);
  ns_product_kernel<T, WHAT><<<(unsigned)tiles, 256, 0, s>>>(o, h, w, step, c, res);
}

// ------------------------------------------------------------------------------------------------ small matrices
// A matrix whose short side fits four 16-row blocks stays in one workgroup's LDS from the first read to the last write: fp32 throughout,
// products on the fp32 matrix instructions, which at these sizes wait for the LDS rather than for each other, and ONE launch for every
// small matrix of a whole list of stacks, where the planes' path needs three launches a step.  Eight waves: a wave takes two of the (up to)
// 16 blocks of S and of P, and half the rows of a 16-column block of X.
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
inline bool is_small(int64_t m, int64_t n) {
  const int64_t s = m < n ? m : n, l = m < n ? n : m;
  return s <= kSmallSide && l <= 4096 && small_lds_bytes(s, l) <= kSmallLds;
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
  if (is_small(m, n)) {
    SmallStacks one;
    one.count = 1;
    one.stack[0] = {src, res, 0, (int)m, (int)n};
    launch_small<T, MOMENTUM>(one, (int)B, small_lds_bytes(m < n ? m : n, m < n ? n : m), steps, c, eps, s);
    PS_CHECK_LAUNCH();
  }
  const Shape h = shape_of(m, n);
  const Work w = work_of(h, B, workspace);
  ns_norm_kernel<T, MOMENTUM><<<dim3(kNormParts, (unsigned)B), 256, 0, s>>>(src, m * n, w.norms);
  // (the columns cover both paddings: rows and columns as given, rounded up to the planes' tiles)
  const int rows = h.tall ? h.lp : h.sp, cols = h.tall ? h.sp : h.lp;
  ns_start_kernel<T, MOMENTUM><<<dim3((unsigned)(cols / 32), (unsigned)(rows / 32), (unsigned)B), 256, 0, s>>>(src, h, w, eps);
  for (int i = 0; i < steps; ++i) {
    launch_product<T, kGram>({w.x, w.x, w.x_plane, w.x_plane, h.s, h.s, h.lp}, h, w, B, i, c, res, s);
    launch_product<T, kPoly>({w.gram, w.gram, w.s_plane, w.s_plane, h.s, h.s, h.sp}, h, w, B, i, c, res, s);
    const Operands apply{w.poly, w.xt[i & 1], w.s_plane, w.xt_plane, h.s, h.l, h.sp};
    if (i + 1 < steps)
      launch_product<T, kApply>(apply, h, w, B, i, c, res, s);
    else
      launch_product<T, kLast>(apply, h, w, B, i, c, res, s);
  }
  PS_CHECK_LAUNCH();
}

constexpr int64_t kMaxSide = 1 << 20;

bool sizes_ok(int64_t B, int64_t m, int64_t n, int steps) {
  return B >= 0 && B <= 65535 && m >= 0 && n >= 0 && m <= kMaxSide && n <= kMaxSide && steps >= 1 && steps <= 64 && (m < n ? m : n) <= 16384 &&
         pair_tiles(m, n, B) < ((int64_t)1 << 31);
}

}  // namespace

extern "C" int64_t ps_newton_schulz_workspace(int64_t B, int64_t m, int64_t n) {
  if (!sizes_ok(B, m, n, 1) || B == 0 || m == 0 || n == 0 || is_small(m, n)) return 0;
  return work_of(shape_of(m, n), B, nullptr).bytes;
}

extern "C" int ps_newton_schulz(const void* g, int64_t B, int64_t m, int64_t n, int dtype, int steps, double a, double b, double c, float grow, float eps, void* out,
                                void* workspace, void* stream) {
  PS_REQUIRE(sizes_ok(B, m, n, steps) && grow >= 1.0f, "ps_newton_schulz: sizes out of range");
  if (B == 0 || m == 0 || n == 0) return 0;
  PS_REQUIRE(g != nullptr && out != nullptr && (workspace != nullptr || is_small(m, n)), "ps_newton_schulz: null argument");
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
    PS_REQUIRE(B[i] * m[i] * n[i] == 0 || (p[i] && g[i] && buf[i] && (workspace || is_small(m[i], n[i]))), "ps_muon_step: null argument");
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
    if (!is_small(m[i], n[i])) {
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
