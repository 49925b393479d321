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

// The 16-byte run of a row that starts at c, without a branch: the last one,
// where less than a run is left, moves back to end with the row, and one that
// would start behind the row takes the same place. The elements that this adds
// are another run's: they are loaded, but neither count nor are stored. A load's
// address then needs no condition, so all loads of a row are under way at once;
// behind branches they wait for each other. Rows narrower than a run (NARROW)
// are taken element by element.
template <typename T, bool NARROW = false>
struct RowRun {
  static constexpr int V = Width<T>::v;
  int c, at, width;

  __device__ __forceinline__ RowRun(int c_, int width_)
      : c(c_), at(NARROW ? c_ : min(c_, width_ - Width<T>::v)), width(width_) {}

  __device__ __forceinline__ bool any() const { return c < width; }
  __device__ __forceinline__ bool whole() const {
    return NARROW ? c + V <= width : at == c;
  }
  __device__ __forceinline__ bool counts(int i) const {
    return NARROW ? c + i < width : at + i >= c;
  }
  // of a row of any type
  template <typename E>
  __device__ __forceinline__ void load(const E* row, float (&o)[V]) const {
    if constexpr (NARROW) load_some<E, V>(row + at, width - at, o, 0.f);
    else load_run<E, V>(row + at, o);
  }
  template <typename E>
  __device__ __forceinline__ void store(E* row, const float (&v)[V]) const {
    if (whole()) {
      store_run<E, V>(row + at, v);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (counts(i)) row[at + i] = (E)v[i];
    }
  }
};

// what a store in T and a load of it give
template <typename T>
__device__ __forceinline__ float rounded(float v) { return (float)(T)v; }

// The value of a lane in the other half of this lane's 2 D lanes, by a move
// between registers: that lane is the one D away for 1 and 2, and the mirrored
// one for 4 and 8, which does as well once the halves agree within themselves.
template <int D>
__device__ __forceinline__ int lane_across(int v) {
  if constexpr (D == 1) return __builtin_amdgcn_update_dpp(v, v, 0xB1, 15, 15, true);
  if constexpr (D == 2) return __builtin_amdgcn_update_dpp(v, v, 0x4E, 15, 15, true);
  if constexpr (D == 4) return __builtin_amdgcn_update_dpp(v, v, 0x141, 15, 15, true);
  return __builtin_amdgcn_update_dpp(v, v, 0x140, 15, 15, true);
}

// f over LANES neighbouring lanes, the same in all of them
template <int LANES, typename F>
__device__ __forceinline__ float lanes_all(float v, F f) {
  if constexpr (LANES > 1) v = f(v, __int_as_float(lane_across<1>(__float_as_int(v))));
  if constexpr (LANES > 2) v = f(v, __int_as_float(lane_across<2>(__float_as_int(v))));
  if constexpr (LANES > 4) v = f(v, __int_as_float(lane_across<4>(__float_as_int(v))));
  if constexpr (LANES > 8) v = f(v, __int_as_float(lane_across<8>(__float_as_int(v))));
  if constexpr (LANES > 16) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_int(v), __float_as_int(v),
                                                    false, false);
    v = f(__int_as_float(r[0]), __int_as_float(r[1]));
  }
  if constexpr (LANES > 32) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_int(v), __float_as_int(v),
                                                    false, false);
    v = f(__int_as_float(r[0]), __int_as_float(r[1]));
  }
  return v;
}

template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  return lanes_all<LANES>(v, [](float a, float b) { return a + b; });
}

template <int LANES>
__device__ __forceinline__ float lanes_max(float v) {
  return lanes_all<LANES>(v, [](float a, float b) { return fmaxf(a, b); });
}

}  // namespace blk
