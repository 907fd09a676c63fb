// 16-byte accesses shared by the kernels that are bound by HBM.
#pragma once
#include "common.cuh"

namespace moe {

static inline bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }

template <typename T> struct Vec { static constexpr int N = 16 / sizeof(T); T v[N]; };

template <typename T>
__device__ __forceinline__ Vec<T> load_vec(const T* p) {
  Vec<T> r;
  *reinterpret_cast<uint4*>(r.v) = *reinterpret_cast<const uint4*>(p);
  return r;
}
template <typename T>
__device__ __forceinline__ void store_vec(T* p, const Vec<T>& r) {
  *reinterpret_cast<uint4*>(p) = *reinterpret_cast<const uint4*>(r.v);
}

}  // namespace moe
