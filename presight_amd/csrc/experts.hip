// Rows sorted by expert and back.  Every one of N rows is assigned to k experts (ids [N,k]; an id outside [0, E) assigns to nobody).
// The N*k assignments, numbered f = n*k + j, are sorted by (expert, f): a stable counting sort, so equal inputs always give equal
// layouts.  The sort is kept both ways round
//     src[p] = f  (sorted place -> assignment, -1 behind the last expert's rows),   dst[f] = p  (assignment -> place, -1: to nobody)
// so that EVERY direction of the exchange is a gather or a one-to-one scatter: no atomics on values, no order that could change sums.
//     dispatch   rows[dst[n,j]] = x[n]                              gradient   dx[n] = sum_j drows[dst[n,j]]      (= combine, w = 1)
//     combine    y[n] = sum_j w[n,j] * rows[dst[n,j]]               gradient   drows[dst[n,j]] = w[n,j] * dy[n],  dw[n,j] = <dy[n], rows[dst[n,j]]>
// All four run over n: x / dy / y are streamed once in order, the k sorted rows are touched as whole rows.  Nothing is computed that
// is not moved, so all of them are bound by HBM.  16384 rows to 8 of 128 experts each, 2048 bf16 features (a large copy reaches 4.9 TB/s),
// one behind the other as a training pass has them, and each repeated by itself:
//     dispatch 604 MB 99 us, 6.1 TB/s, and 118 | combine 604 MB 152 us, 4.0 TB/s, and 123 | combine's gradients 1141 MB 245 us, 4.7 TB/s |
//     the plan of 131072 assignments 15 us
// One row after the other, each fetched whole, is best: four or eight rows of an assignment's at once were a tenth to a half slower.
// 65536 rows to 2 of 16, 64 fp32 features: 10 us and less for 50 MB, 17 us for 84; one row: 2 us each and 4 for its plan, all latency.
#include "common.hpp"
#include "expert_types.hpp"

namespace {

using namespace ps;

constexpr int kPlanThreads = 1024;
constexpr int kPlanWaves = kPlanThreads / 64;
constexpr int kPlanOneBlock = 8192;   // assignments one workgroup sorts alone (one launch instead of two)
constexpr int kPlanMaxBlocks = 128;   // every placing workgroup sums the counts of all counting workgroups

__device__ __forceinline__ int load_id(const void* ids, int wide, int64_t f, int E) {
  const int64_t v = wide ? reinterpret_cast<const int64_t*>(ids)[f] : (int64_t)reinterpret_cast<const int*>(ids)[f];
  return v >= 0 && v < E ? (int)v : -1;
}

// lanes of the wave that hold the same id (id < 2^bits, lanes with valid = false match nobody)
__device__ __forceinline__ unsigned long long same_id(int id, bool valid, int bits) {
  unsigned long long m = __ballot(valid);
  for (int b = 0; b < bits; ++b) {
    const unsigned long long v = __ballot((id >> b) & 1);
    m &= ((id >> b) & 1) ? v : ~v;
  }
  return valid ? m : 0ull;
}

__global__ __launch_bounds__(kPlanThreads) void plan_count_kernel(const void* __restrict__ ids, int wide, int64_t M, int E, int64_t chunk,
                                                                  int* __restrict__ hist) {
  extern __shared__ int cnt[];  // [E]
  for (int e = threadIdx.x; e < E; e += kPlanThreads) cnt[e] = 0;
  __syncthreads();
  const int64_t f0 = blockIdx.x * chunk, f1 = f0 + chunk < M ? f0 + chunk : M;
  for (int64_t f = f0 + threadIdx.x; f < f1; f += kPlanThreads) {
    const int id = load_id(ids, wide, f, E);
    if (id >= 0) atomicAdd(&cnt[id], 1);
  }
  __syncthreads();
  for (int e = threadIdx.x; e < E; e += kPlanThreads) hist[(int64_t)blockIdx.x * E + e] = cnt[e];
}

// 131072 assignments: 5 us to count and 10 to place them, neither near a limit of the memory: a workgroup's two passes over its ids, the
// second one's ranks, and the scans between them wait for each other.
// One workgroup places the assignments [f0, f0 + chunk).  Each wave owns a contiguous run of them and counts it by itself (cnt[wave][e],
// ballots instead of atomics: the rank inside a 64-wide round is a popcount), the counts become first places by a scan over waves, the
// workgroups before this one (hist) and the experts, and a second pass over the same ids hands the places out in order.
__global__ __launch_bounds__(kPlanThreads) void plan_place_kernel(const void* __restrict__ ids, int wide, int64_t M, int E, int bits, int64_t chunk,
                                                                  const int* __restrict__ hist, int* __restrict__ offsets, int* __restrict__ src,
                                                                  int* __restrict__ dst) {
  extern __shared__ int sh[];
  int* cnt = sh;                       // [waves][E]
  int* total = sh + kPlanWaves * E;    // [E] rows of expert e in all workgroups
  int* before = total + E;             // [E] ... in the workgroups before this one
  __shared__ int wave_sum[kPlanWaves];
  const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
  for (int i = threadIdx.x; i < (kPlanWaves + 2) * E; i += kPlanThreads) sh[i] = 0;
  __syncthreads();
  const int64_t seg = chunk / kPlanWaves;  // (a multiple of 64)
  const int64_t f0 = blockIdx.x * chunk + wave * seg;
  const unsigned long long below = (1ull << lane) - 1ull;
  for (int64_t r = 0; r < seg && f0 + r < M; r += 64) {
    const int64_t f = f0 + r + lane;
    const int id = f < M ? load_id(ids, wide, f, E) : -1;
    const unsigned long long m = same_id(id, id >= 0, bits);
    if (id >= 0 && (m & below) == 0ull) cnt[wave * E + id] += __popcll(m);
  }
  if (hist != nullptr) {
    // (expert, part) per thread: the parts of one expert's column are summed side by side
    const int width = 1 << bits, parts = kPlanThreads / width > 0 ? kPlanThreads / width : 1;
    const int part = threadIdx.x / width;
    for (int e = threadIdx.x % width; e < E && part < parts; e += kPlanThreads) {
      int all = 0, prev = 0;
      for (int b = part; b < (int)gridDim.x; b += parts) {
        const int h = hist[(int64_t)b * E + e];
        all += h;
        if (b < (int)blockIdx.x) prev += h;
      }
      atomicAdd(&total[e], all);
      atomicAdd(&before[e], prev);
    }
  }
  __syncthreads();
  const int e = threadIdx.x;  // E <= kPlanThreads
  int mine = 0, first = 0;
  if (e < E) {
    int run = 0;
    for (int w = 0; w < kPlanWaves; ++w) {
      const int c = cnt[w * E + e];
      cnt[w * E + e] = run;
      run += c;
    }
    mine = hist != nullptr ? total[e] : run;
  }
  int incl = mine;
  for (int d = 1; d < 64; d <<= 1) {
    const int o = __shfl_up(incl, d, 64);
    if (lane >= d) incl += o;
  }
  if (lane == 63) wave_sum[wave] = incl;
  __syncthreads();
  for (int w = 0; w < wave; ++w) first += wave_sum[w];
  int held = 0;
  for (int w = 0; w < kPlanWaves; ++w) held += wave_sum[w];
  first += incl - mine;
  if (e < E) {
    const int start = first + before[e];
    for (int w = 0; w < kPlanWaves; ++w) cnt[w * E + e] += start;
    if (blockIdx.x == 0) offsets[e] = first;
  }
  if (blockIdx.x == 0 && threadIdx.x == 0) offsets[E] = held;
  __syncthreads();
  for (int64_t r = 0; r < seg && f0 + r < M; r += 64) {
    const int64_t f = f0 + r + lane;
    const int id = f < M ? load_id(ids, wide, f, E) : -1;
    const unsigned long long m = same_id(id, id >= 0, bits);
    if (id >= 0) {
      const int p = cnt[wave * E + id] + __popcll(m & below);
      src[p] = (int)f;
      dst[f] = p;
    } else if (f < M) {
      dst[f] = -1;
    }
    __builtin_amdgcn_wave_barrier();
    if (id >= 0 && (m & below) == 0ull) cnt[wave * E + id] += __popcll(m);
    __builtin_amdgcn_wave_barrier();
    if (f < M && f >= held) src[f] = -1;  // (this lane's number taken as a sorted place)
  }
}

// ------------------------------------------------------------------------------------------------ rows
// G lanes work on one row in steps of VEC elements (16 bytes, of rows that have them): a 256-byte row keeps 16 lanes busy, so 4 rows share a
// wave; long rows take a whole wave.  Rows may start at any element; the last step of one that is no whole number of them starts early,
// over elements that come out the same twice.  (10007 rows to 3 of 37, 195 fp16, with gradients: 28 us; 64 element by element.)
__device__ __forceinline__ int step_at(int c, int D, int vec) { return c + vec <= D ? c : D - vec; }

template <typename T, int VEC>
__global__ __launch_bounds__(256) void dispatch_kernel(const T* __restrict__ x, int64_t x_stride, const int* __restrict__ dst,
                                                       const int* __restrict__ held, int64_t N, int k, int D, int G, T* __restrict__ rows) {
  const int l = threadIdx.x & (G - 1);
  const int64_t places = N * k, total = *held;
  for (int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G; n < N; n += (int64_t)gridDim.x * 256 / G) {
    const int* d = dst + n * k;
    for (int u = l * VEC; u < D; u += G * VEC) {
      const int c = step_at(u, D, VEC);
      const Pack<T, VEC> v = load_any<T, VEC>(x + n * x_stride + c);
      for (int j = 0; j < k; ++j) {
        const int p = d[j];
        if (p >= 0 && p < places) store_any(rows + (int64_t)p * D + c, v);
      }
    }
    for (int j = 0; j < k; ++j) {  // the places behind the last expert's rows are shared out over the same lanes
      const int64_t p = n * k + j;
      if (p >= total)
        for (int u = l * VEC; u < D; u += G * VEC) store_any(rows + p * D + step_at(u, D, VEC), Pack<T, VEC>{});
    }
  }
}

// y[n] = sum_j w[n,j] * rows[dst[n,j]] in fp32, rounded once; w == nullptr: all ones.  A weight or a row of an assignment to nobody is
// never read.
template <typename T, int VEC>
__global__ __launch_bounds__(256) void combine_kernel(const T* __restrict__ rows, int64_t r_stride, const float* __restrict__ w,
                                                      const int* __restrict__ dst, int64_t N, int k, int D, int G, T* __restrict__ y) {
  const int l = threadIdx.x & (G - 1);
  const int64_t places = N * k;
  for (int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G; n < N; n += (int64_t)gridDim.x * 256 / G) {
    const int* d = dst + n * k;
    for (int u = l * VEC; u < D; u += G * VEC) {
      const int c = step_at(u, D, VEC);
      float acc[VEC] = {};
      for (int j = 0; j < k; ++j) {
        const int p = d[j];
        if (p < 0 || p >= places) continue;
        const Pack<T, VEC> v = load_any<T, VEC>(rows + p * r_stride + c);
        const float wj = w != nullptr ? w[n * k + j] : 1.0f;
#pragma unroll
        for (int i = 0; i < VEC; ++i) acc[i] = fmaf(wj, to_f32(v.v[i]), acc[i]);
      }
      Pack<T, VEC> o;
#pragma unroll
      for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(acc[i]);
      store_any(y + n * D + c, o);
    }
  }
}

// both gradients of combine in one pass over the sorted rows; drows / dw may be null (not asked for).  (More than a wave on one row, its
// products joined in LDS: 260 us for 245.)
template <typename T, int VEC>
__global__ __launch_bounds__(256) void combine_bwd_kernel(const T* __restrict__ dy, int64_t dy_stride, const T* __restrict__ rows, int64_t r_stride,
                                                          const float* __restrict__ w, const int* __restrict__ dst, const int* __restrict__ held,
                                                          int64_t N, int k, int D, int G, T* __restrict__ drows, float* __restrict__ dw) {
  const int l = threadIdx.x & (G - 1);
  const int64_t places = N * k, total = *held;
  for (int64_t n = ((int64_t)blockIdx.x * 256 + threadIdx.x) / G; n < N; n += (int64_t)gridDim.x * 256 / G) {  // (a row's lanes stay together)
    for (int j = 0; j < k; ++j) {
      const int p = dst[n * k + j];
      float dot = 0.0f;
      if (p >= 0 && p < places) {
        const float wj = w[n * k + j];
        for (int u = l * VEC; u < D; u += G * VEC) {
          const int c = step_at(u, D, VEC);
          const Pack<T, VEC> g = load_any<T, VEC>(dy + n * dy_stride + c);
          if (dw != nullptr) {
            const Pack<T, VEC> r = load_any<T, VEC>(rows + p * r_stride + c);
#pragma unroll
            for (int i = 0; i < VEC; ++i) {
              const float sum = fmaf(to_f32(g.v[i]), to_f32(r.v[i]), dot);
              dot = c + i >= u ? sum : dot;  // (once each)
            }
          }
          if (drows != nullptr) {
            Pack<T, VEC> o;
#pragma unroll
            for (int i = 0; i < VEC; ++i) o.v[i] = from_f32<T>(wj * to_f32(g.v[i]));
            store_any(drows + (int64_t)p * D + c, o);
          }
        }
      }
      if (dw != nullptr) {
        for (int s = G >> 1; s > 0; s >>= 1) dot += __shfl_xor(dot, s, 64);
        if (l == 0) dw[n * k + j] = dot;
      }
      const int64_t q = n * k + j;
      if (drows != nullptr && q >= total)
        for (int u = l * VEC; u < D; u += G * VEC) store_any(drows + q * D + step_at(u, D, VEC), Pack<T, VEC>{});
    }
  }
}

// elements a lane moves at a time: 16 bytes, fewer where a row has not got them
int vec_elems(int size, int64_t D) {
  int v = 16 / size;
  while (v > 1 && v > D) v >>= 1;
  return v;
}

// most: 64 where a row's lanes add up (one wave), else a workgroup: a row of 4 KiB is fetched whole rather than in four visits (combine,
// 16384 rows of 8 x 2048 bf16: 156 -> 127 us)
int lanes_per_row(int64_t D, int vec, int most) {
  const int64_t units = (D + vec - 1) / vec;
  int g = 1;
  while (g < most && g < units) g <<= 1;
  return g;
}

template <typename F>
int by_type(int dtype, F&& f) {
  if (dtype == kF32) return f(float{});
  if (dtype == kF16) return f(_Float16{});
  if (dtype == kBF16) return f(__bf16{});
  ps_set_error("unknown element type (0 fp32, 1 fp16, 2 bf16)");
  return -1;
}

#define PS_BY_VEC(T, vec, CALL)                                 \
  do {                                                          \
    if constexpr (sizeof(T) == 2) {                             \
      if ((vec) == 8) { constexpr int VEC = 8; CALL; break; }   \
    }                                                           \
    if ((vec) == 4) { constexpr int VEC = 4; CALL; break; }     \
    if ((vec) == 2) { constexpr int VEC = 2; CALL; break; }     \
    { constexpr int VEC = 1; CALL; }                            \
  } while (0)

bool fits(int64_t N, int k, int64_t D) { return N >= 0 && k >= 1 && D >= 0 && D < (1 << 28) && N < ((int64_t)1 << 31) / k; }

}  // namespace

extern "C" int64_t ps_expert_plan_workspace(int64_t M, int E) {
  return M <= kPlanOneBlock || E < 1 ? 0 : (int64_t)kPlanMaxBlocks * E;
}

extern "C" int ps_expert_plan(const void* ids, int ids_are_64, int64_t M, int E, int32_t* offsets, int32_t* src, int32_t* dst, int32_t* workspace,
                              void* stream) {
  PS_REQUIRE(E >= 1 && E <= kPlanThreads, "ps_expert_plan: 1..1024 experts");
  PS_REQUIRE(M >= 0 && M < ((int64_t)1 << 31) - (1 << 20), "ps_expert_plan: the assignments must fit 32-bit places");
  PS_REQUIRE(offsets != nullptr && (M == 0 || (ids != nullptr && src != nullptr && dst != nullptr)), "ps_expert_plan: null argument");
  PS_REQUIRE(M <= kPlanOneBlock || workspace != nullptr, "ps_expert_plan: needs its workspace (ps_expert_plan_workspace)");
  hipStream_t s = (hipStream_t)stream;
  int bits = 0;
  while ((1 << bits) < E) ++bits;
  const size_t lds = (size_t)(kPlanWaves + 2) * E * sizeof(int);
  if (lds > 64 * 1024) hipFuncSetAttribute((const void*)plan_place_kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)lds);
  if (M <= kPlanOneBlock) {
    const int64_t chunk = ((M + kPlanThreads - 1) / kPlanThreads) * kPlanThreads;
    plan_place_kernel<<<1, kPlanThreads, lds, s>>>(ids, ids_are_64, M, E, bits, chunk, nullptr, offsets, src, dst);
    PS_CHECK_LAUNCH();
  }
  int64_t chunk = 2048;
  if (M > chunk * kPlanMaxBlocks) chunk = ((M + kPlanMaxBlocks - 1) / kPlanMaxBlocks + kPlanThreads - 1) / kPlanThreads * kPlanThreads;
  const unsigned blocks = (unsigned)((M + chunk - 1) / chunk);
  plan_count_kernel<<<blocks, kPlanThreads, (size_t)E * sizeof(int), s>>>(ids, ids_are_64, M, E, chunk, workspace);
  plan_place_kernel<<<blocks, kPlanThreads, lds, s>>>(ids, ids_are_64, M, E, bits, chunk, workspace, offsets, src, dst);
  PS_CHECK_LAUNCH();
}

extern "C" int ps_expert_dispatch(const void* x, int64_t x_stride, const int32_t* dst, const int32_t* held, int64_t N, int k, int64_t D, int dtype,
                                  void* rows, void* stream) {
  PS_REQUIRE(fits(N, k, D), "ps_expert_dispatch: sizes out of range");
  if (N == 0 || D == 0) return 0;
  PS_REQUIRE(x != nullptr && dst != nullptr && held != nullptr && rows != nullptr, "ps_expert_dispatch: null argument");
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int vec = vec_elems(sizeof(T), D), G = lanes_per_row(D, vec, 256);
    const unsigned blocks = blocks_of_256(N * G);
    PS_BY_VEC(T, vec, (dispatch_kernel<T, VEC><<<blocks, 256, 0, (hipStream_t)stream>>>((const T*)x, x_stride, dst, held, N, k, (int)D, G, (T*)rows)));
    PS_CHECK_LAUNCH();
  });
}

extern "C" int ps_expert_combine(const void* rows, int64_t rows_stride, const float* weights, const int32_t* dst, int64_t N, int k, int64_t D,
                                 int dtype, void* y, void* stream) {
  PS_REQUIRE(fits(N, k, D), "ps_expert_combine: sizes out of range");
  if (N == 0 || D == 0) return 0;
  PS_REQUIRE(rows != nullptr && dst != nullptr && y != nullptr, "ps_expert_combine: null argument");
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int vec = vec_elems(sizeof(T), D), G = lanes_per_row(D, vec, 256);
    const unsigned blocks = blocks_of_256(N * G);
    PS_BY_VEC(T, vec, (combine_kernel<T, VEC><<<blocks, 256, 0, (hipStream_t)stream>>>((const T*)rows, rows_stride, weights, dst, N, k, (int)D, G, (T*)y)));
    PS_CHECK_LAUNCH();
  });
}

extern "C" int ps_expert_combine_bwd(const void* dy, int64_t dy_stride, const void* rows, int64_t rows_stride, const float* weights,
                                     const int32_t* dst, const int32_t* held, int64_t N, int k, int64_t D, int dtype, void* drows, float* dw,
                                     void* stream) {
  PS_REQUIRE(fits(N, k, D), "ps_expert_combine_bwd: sizes out of range");
  if (N == 0 || (drows == nullptr && dw == nullptr)) return 0;
  PS_REQUIRE(weights != nullptr && dst != nullptr && held != nullptr && (D == 0 || (dy != nullptr && rows != nullptr)), "ps_expert_combine_bwd: null argument");
  return by_type(dtype, [&](auto zero) {
    using T = decltype(zero);
    const int vec = vec_elems(sizeof(T), D), G = lanes_per_row(D, vec, 64);
    const unsigned blocks = blocks_of_256(N * G);
    PS_BY_VEC(T, vec, (combine_bwd_kernel<T, VEC><<<blocks, 256, 0, (hipStream_t)stream>>>((const T*)dy, dy_stride, (const T*)rows, rows_stride, weights,
                                                                                           dst, held, N, k, (int)D, G, (T*)drows, dw)));
    PS_CHECK_LAUNCH();
  });
}
