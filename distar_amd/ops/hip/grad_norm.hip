// The norm of many tensors together, and their scaling to a largest norm.
//
//   n = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|
//   g *= min(1, max_norm / (n + eps))
//
// Memory bounds both: the norm reads every value once, the scaling reads and
// writes each once more, and not at all in place when nothing is clipped. The
// tensors' addresses and sizes travel in the kernel's arguments, some hundred
// tensors a launch, so no table is copied to the device and a captured graph
// keeps its own. A block takes one chunk of one tensor and leaves one partial
// sum; a last block adds those up in a fixed order. Sums are 64-bit: squares
// of any 32-bit value fit, and the conversion hides behind the loads.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr int kThreads = 256;
constexpr int kTensors = 112;     // 112 x (8 + 8 + 8 + 4 + 1 + 1) < 4 KB

struct Table {
  const void* in[kTensors];
  void* out[kTensors];
  int64_t numel[kTensors];
  uint32_t first[kTensors];       // the tensor's first block in this launch
  uint8_t in_dtype[kTensors], out_dtype[kTensors];
  int count;
};

// which tensor a block belongs to
__device__ __forceinline__ int find(const Table& t, uint32_t block) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// ORDER 0 stands for the largest absolute value. That is taken on the bits,
// where every NaN is above infinity, so that one stays visible.
template <typename T, int ORDER>
__device__ __forceinline__ double norm_part(const T* p, int64_t n) {
  constexpr int V = Width<T>::v;
  double acc[2] = {0., 0.};
  uint32_t most = 0;
  for (int64_t i = (int64_t)threadIdx.x * V; i < n; i += kThreads * V) {
    float v[V];
    load_some<T, V>(p + i, (int)(n - i < V ? n - i : V), v, 0.f);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      if constexpr (ORDER == 2) {
        acc[j & 1] = fma((double)v[j], (double)v[j], acc[j & 1]);
      } else if constexpr (ORDER == 1) {
        acc[j & 1] += (double)fabsf(v[j]);
      } else {
        const uint32_t b = __float_as_uint(v[j]) & 0x7fffffffu;
        most = b > most ? b : most;
      }
    }
  }
  return ORDER ? acc[0] + acc[1] : (double)__uint_as_float(most);
}

template <int ORDER>
__device__ __forceinline__ double both(double a, double b) {
  if constexpr (ORDER) return a + b;
  return a != a ? a : (b > a || b != b) ? b : a;
}

template <int ORDER, int THREADS>
__device__ __forceinline__ double block_all(double v, double* lds) {
#pragma unroll
  for (int o = 1; o < 64; o <<= 1) v = both<ORDER>(v, __shfl_xor(v, o, 64));
  if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
  __syncthreads();
  if (threadIdx.x == 0)
    for (int w = 1; w < THREADS / 64; ++w) v = both<ORDER>(v, lds[w]);
  return v;
}

template <int ORDER>
__global__ __launch_bounds__(kThreads) void norm_kernel(Table t, int64_t chunk,
                                                        double* partial) {
  __shared__ double lds[kThreads / 64];
  const int k = find(t, blockIdx.x);
  const int64_t at = (int64_t)(blockIdx.x - t.first[k]) * chunk;
  const int64_t left = t.numel[k] - at;
  const int64_t n = left < chunk ? left : chunk;
  double v;
  if (t.in_dtype[k] == kF32)
    v = norm_part<float, ORDER>((const float*)t.in[k] + at, n);
  else if (t.in_dtype[k] == kBF16)
    v = norm_part<bf16, ORDER>((const bf16*)t.in[k] + at, n);
  else
    v = norm_part<f16, ORDER>((const f16*)t.in[k] + at, n);
  v = block_all<ORDER, kThreads>(v, lds);
  if (threadIdx.x == 0) partial[blockIdx.x] = v;
}

template <int ORDER>
__global__ __launch_bounds__(1024) void norm_join_kernel(
    const double* partial, int64_t blocks, float* norm, float* coef,
    float max_norm, float eps) {
  __shared__ double lds[16];
  double v = 0.;
  for (int64_t i = threadIdx.x; i < blocks; i += 1024)
    v = both<ORDER>(v, partial[i]);
  v = block_all<ORDER, 1024>(v, lds);
  if (threadIdx.x == 0) {
    const float n = (float)(ORDER == 2 ? sqrt(v) : v);
    *norm = n;
    const float c = max_norm / (n + eps);
    *coef = c > 1.f ? 1.f : c;              // a NaN stays one
  }
}

template <typename T, typename O>
__device__ __forceinline__ void scale_part(const T* p, O* q, int64_t n, float c) {
  constexpr int V = Width<T>::v;
  for (int64_t i = (int64_t)threadIdx.x * V; i < n; i += kThreads * V) {
    const int some = (int)(n - i < V ? n - i : V);
    float v[V];
    load_some<T, V>(p + i, some, v, 0.f);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] *= c;
    store_some<O, V>(q + i, some, v);
  }
}

template <typename T>
__device__ __forceinline__ void scale_to(const Table& t, int k, int64_t at,
                                         int64_t n, float c) {
  const T* p = (const T*)t.in[k] + at;
  if (t.out_dtype[k] == kF32)
    scale_part<T, float>(p, (float*)t.out[k] + at, n, c);
  else if (t.out_dtype[k] == kBF16)
    scale_part<T, bf16>(p, (bf16*)t.out[k] + at, n, c);
  else
    scale_part<T, f16>(p, (f16*)t.out[k] + at, n, c);
}

__global__ __launch_bounds__(kThreads) void scale_kernel(Table t, int64_t chunk,
                                                         const float* coef) {
  const float c = *coef;
  const int k = find(t, blockIdx.x);
  if (c == 1.f && t.in[k] == t.out[k]) return;
  const int64_t at = (int64_t)(blockIdx.x - t.first[k]) * chunk;
  const int64_t left = t.numel[k] - at;
  const int64_t n = left < chunk ? left : chunk;
  if (t.in_dtype[k] == kF32) scale_to<float>(t, k, at, n, c);
  else if (t.in_dtype[k] == kBF16) scale_to<bf16>(t, k, at, n, c);
  else scale_to<f16>(t, k, at, n, c);
}

// fills a table from tensor i on; returns the blocks it takes
uint32_t fill(const GradTensor* g, int count, int64_t chunk, int& i, Table& t) {
  uint32_t blocks = 0;
  t.count = 0;
  for (; i < count && t.count < kTensors; ++i) {
    if (!g[i].numel) continue;
    const int k = t.count++;
    t.in[k] = g[i].in;
    t.out[k] = g[i].out;
    t.numel[k] = g[i].numel;
    t.in_dtype[k] = (uint8_t)g[i].in_dtype;
    t.out_dtype[k] = (uint8_t)g[i].out_dtype;
    t.first[k] = blocks;
    blocks += (uint32_t)((g[i].numel + chunk - 1) / chunk);
  }
  return blocks;
}

}  // namespace

int64_t grad_norm_blocks(const GradTensor* g, int count, int64_t* chunk) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += g[i].numel;
  int64_t c = 16384;
  while (total / c > 16384) c *= 2;
  *chunk = c;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i) blocks += (g[i].numel + c - 1) / c;
  return blocks;
}

void grad_norm(const GradTensor* g, int count, int64_t chunk, int order,
               double* partial, int64_t blocks, float* norm, float* coef,
               float max_norm, float eps, hipStream_t stream) {
  Table t;
  double* at = partial;
  for (int i = 0; i < count;) {
    const uint32_t n = fill(g, count, chunk, i, t);
    if (!n) break;
    if (order == 2) norm_kernel<2><<<n, kThreads, 0, stream>>>(t, chunk, at);
    else if (order == 1) norm_kernel<1><<<n, kThreads, 0, stream>>>(t, chunk, at);
    else norm_kernel<0><<<n, kThreads, 0, stream>>>(t, chunk, at);
    at += n;
  }
  if (order == 2)
    norm_join_kernel<2><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
  else if (order == 1)
    norm_join_kernel<1><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
  else
    norm_join_kernel<0><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
}

void grad_scale(const GradTensor* g, int count, int64_t chunk,
                const float* coef, hipStream_t stream) {
  Table t;
  for (int i = 0; i < count;) {
    const uint32_t n = fill(g, count, chunk, i, t);
    if (!n) break;
    scale_kernel<<<n, kThreads, 0, stream>>>(t, chunk, coef);
  }
}

}  // namespace blk
