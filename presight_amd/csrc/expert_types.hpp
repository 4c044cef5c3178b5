// Element types of the expert and matrix-update operators (fp32, fp16, bf16) and rows read and written in packs of them.
#pragma once
#include <initializer_list>
#include "common.hpp"

namespace ps {

enum : int { kF32 = 0, kF16 = 1, kBF16 = 2 };

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(_Float16 v) { return (float)v; }
__device__ __forceinline__ float to_f32(__bf16 v) { return (float)v; }
template <typename T>
__device__ __forceinline__ T from_f32(float v) {  // round to nearest even
  return (T)v;
}

// A launch holds fewer than 2^32 threads: workgroups of 256 for n of them, which take more than one each beyond 2^31
constexpr int64_t kMaxThreads = (int64_t)1 << 32;
inline unsigned blocks_of_256(int64_t n) { return (unsigned)((n < kMaxThreads / 2 ? n + 255 : kMaxThreads / 2) / 256); }

template <typename T, int VEC>
struct alignas(sizeof(T) * VEC) Pack {
  T v[VEC];
};
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_pack(const T* p) {
  return *reinterpret_cast<const Pack<T, VEC>*>(p);
}
template <typename T, int VEC>
__device__ __forceinline__ void store_pack(T* p, const Pack<T, VEC>& v) {
  *reinterpret_cast<Pack<T, VEC>*>(p) = v;
}
// ... at any element's address (one access all the same: the memory takes 16 bytes at any address, and splits what crosses a line)
template <typename T, int VEC>
__device__ __forceinline__ Pack<T, VEC> load_any(const T* p) {
  Pack<T, VEC> v;
  __builtin_memcpy(&v, p, sizeof v);
  return v;
}
template <typename T, int VEC>
__device__ __forceinline__ void store_any(T* p, const Pack<T, VEC>& v) {
  __builtin_memcpy(p, &v, sizeof v);
}

}  // namespace ps
