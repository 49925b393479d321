// What the kernels around the policy transformer share: element types, loads
// and stores of short runs of elements, and sums over the lanes of a wave.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

namespace blk {

using bf16 = __bf16;
using f16 = _Float16;

// elements that fill 16 bytes
template <typename T> struct Width { static constexpr int v = 16 / sizeof(T); };

// A run of V elements from an address aligned to one element only: global
// memory takes a 16-byte access at any element's address, so odd widths and
// views need no path of their own.
template <typename T, int V>
__device__ __forceinline__ void load_run(const T* p, float (&o)[V]) {
  T t[V];
  __builtin_memcpy(t, p, sizeof(t));
#pragma unroll
  for (int i = 0; i < V; ++i) o[i] = (float)t[i];
}

template <typename T, int V>
__device__ __forceinline__ void store_run(T* p, const float (&v)[V]) {
  T t[V];
#pragma unroll
  for (int i = 0; i < V; ++i) t[i] = (T)v[i];
  __builtin_memcpy(p, t, sizeof(t));
}

// the same for a run of which only the first n elements exist
template <typename T, int V>
__device__ __forceinline__ void load_some(const T* p, int n, float (&o)[V],
                                          float fill) {
  if (n >= V) {
    load_run<T, V>(p, o);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) o[i] = i < n ? (float)p[i] : fill;
  }
}

template <typename T, int V>
__device__ __forceinline__ void store_some(T* p, int n, const float (&v)[V]) {
  if (n >= V) {
    store_run<T, V>(p, v);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n) p[i] = (T)v[i];
  }
}

// what a store in T and a load of it give
template <typename T>
__device__ __forceinline__ float rounded(float v) { return (float)(T)v; }

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v += __shfl_xor(v, o, 64);
  return v;
}

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
#pragma unroll
  for (int o = 1; o < LANES; o <<= 1) v = fmaxf(v, __shfl_xor(v, o, 64));
  return v;
}

}  // namespace blk
