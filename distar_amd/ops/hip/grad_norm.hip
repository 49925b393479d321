// The norm of many tensors together, and their scaling to a largest norm.
//
//   n = (sum |g|^p)^(1/p), p = 1 or 2, or max |g|
//   g *= min(1, max_norm / (n + eps))
//
// Memory bounds both: the norm reads every value once, the scaling reads and
// writes each once more, and not at all in place when nothing is clipped. The
// tensors' addresses and sizes travel in the kernel's arguments (4 KB hold some
// 230 tensors, or 160 with outputs; neighbours in memory count as one), so no table
// is copied to the device and a captured graph keeps its own. A block takes one
// chunk of one tensor and leaves one partial sum; a last block adds those up in a
// fixed order. Sums over more than 8 elements are 64-bit, so they neither overflow
// nor drift. Which elements share a run, and so the sums' last digits, depends on where
// the tensors lie: chunks begin at 16-byte boundaries, and neighbours are one tensor.
// The same call on the same memory gives the same norm; equal values that lie
// otherwise may differ in its last bit.
//
// Tensors may start at any element (views of a flat bucket do). A chunk is cut
// where 16-byte accesses are aligned: to what is read in the norm, to what is
// written in the scaling, where the other side then is not; unaligned reads cost
// little, unaligned writes half the rate.
//
// 170 M bf16 values end to end, scaled into fp32: norm 94 us (3.6 TB/s; a large
// sum reads 4.0), join 5 us, scaling 167 us (6.1 TB/s over reads and writes). 56 M
// fp32 values in 332 tensors, not clipped: 39 us in two launches, join 5 us, and
// 6 us for the scaling to find that there is nothing to do.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr int kThreads = 256;
constexpr int kRun = 8;                       // elements a thread takes at once
constexpr int kUnder = 4;                     // runs under way together
constexpr int kPass = kThreads * kRun * kUnder;

template <bool OUT>
struct Table {
  static constexpr int most = OUT ? 160 : 232;
  const void* in[most];
  void* out[OUT ? most : 1];
  uint32_t numel[most];
  uint32_t first[most];           // the tensor's first block in this launch
  uint8_t dtype[most];            // in + 4 out
  int count;
};
static_assert(sizeof(Table<false>) <= 4000 && sizeof(Table<true>) <= 4024, "arguments");

// which tensor a block belongs to
template <bool OUT>
__device__ __forceinline__ int find(const Table<OUT>& t, uint32_t block) {
  int lo = 0, hi = t.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= block) lo = mid; else hi = mid - 1;
  }
  return lo;
}

// Elements of T before the first 16-byte boundary.
template <typename T>
__device__ __forceinline__ uint32_t to_boundary(const T* p) {
  return (uint32_t)(-(uintptr_t)p & 15) / sizeof(T);
}

// The part [begin, end) of a tensor of n elements that a block takes: chunks
// from the first boundary on, the elements before it with the first.
struct Part {
  uint32_t head, begin, end;      // [0, head) too, for the first chunk
  __device__ __forceinline__ Part(uint32_t n, uint32_t boundary, uint32_t index,
                                  uint32_t chunk) {
    boundary = boundary < n ? boundary : n;
    head = index ? 0 : boundary;
    const uint64_t from = boundary + (uint64_t)index * chunk, to = from + chunk;
    begin = from < n ? (uint32_t)from : n;
    end = to < n ? (uint32_t)to : n;
  }
};

// ORDER 0 stands for the largest absolute value. That is taken on the bits,
// where every NaN is above infinity, so that one stays visible.
// A run of 8 is summed in 32 bits, by a tree (an error of at most 4 roundings of
// its sum of squares, 2 of half its sum), and added to a 64-bit sum: a conversion
// and an addition of 64 bits a run instead of two an element. Runs whose squares
// could leave the 32-bit range on either side go element by element.
template <int ORDER>
struct Acc {
  double sum[2] = {0., 0.};
  uint32_t most = 0;

  __device__ __forceinline__ void add(float v) {
    if constexpr (ORDER == 2) sum[0] = fma((double)v, (double)v, sum[0]);
    else if constexpr (ORDER == 1) sum[0] += (double)fabsf(v);
    else most = max(most, __float_as_uint(v) & 0x7fffffffu);
  }
  __device__ __forceinline__ void add(const float (&v)[kRun]) {
    if constexpr (ORDER == 0) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) add(v[j]);
      return;
    }
    float m = 0.f;
#pragma unroll
    for (int j = 0; j < kRun; ++j) m = fmaxf(m, fabsf(v[j]));
    if (ORDER == 2 ? (m <= 1e18f && m >= 1e-14f) || m == 0.f : m <= 1e37f) {
      float s[kRun / 2];
#pragma unroll
      for (int j = 0; j < kRun / 2; ++j)
        s[j] = ORDER == 2 ? fmaf(v[2 * j], v[2 * j], v[2 * j + 1] * v[2 * j + 1])
                          : fabsf(v[2 * j]) + fabsf(v[2 * j + 1]);
      if constexpr (ORDER == 2) {
        sum[0] += (double)((s[0] + s[1]) + (s[2] + s[3]));
      } else {
        sum[0] += (double)(s[0] + s[1]);
        sum[1] += (double)(s[2] + s[3]);
      }
    } else {
#pragma unroll 1
      for (int j = 0; j < kRun; ++j) {
        float x = v[0];               // v[j] without memory
#pragma unroll
        for (int k = 1; k < kRun; ++k) x = j == k ? v[k] : x;
        add(x);
      }
    }
  }
  __device__ __forceinline__ double value() const {
    return ORDER ? sum[0] + sum[1] : (double)__uint_as_float(most);
  }
};

template <typename T, int ORDER>
__device__ __forceinline__ double norm_part(const T* p, uint32_t n, uint32_t index,
                                            uint32_t chunk) {
  const Part part(n, to_boundary(p), index, chunk);
  Acc<ORDER> acc;
  if (threadIdx.x < part.head) acc.add((float)p[threadIdx.x]);
  uint32_t i = part.begin;
  for (; part.end - i >= kPass; i += kPass) {
    float v[kUnder][kRun];
#pragma unroll
    for (int k = 0; k < kUnder; ++k)
      load_run<T, kRun>(p + i + (k * kThreads + threadIdx.x) * kRun, v[k]);
#pragma unroll
    for (int k = 0; k < kUnder; ++k) acc.add(v[k]);
  }
  for (i += threadIdx.x * kRun; i < part.end; i += kThreads * kRun) {
    float v[kRun];
    load_some<T, kRun>(p + i, (int)(part.end - i), v, 0.f);
    acc.add(v);
  }
  return acc.value();
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
__global__ __launch_bounds__(kThreads) void norm_kernel(Table<false> t,
                                                        uint32_t chunk,
                                                        double* partial) {
  __shared__ double lds[kThreads / 64];
  const int k = find(t, blockIdx.x);
  const uint32_t index = blockIdx.x - t.first[k], n = t.numel[k];
  double v;
  if ((t.dtype[k] & 3) == kF32)
    v = norm_part<float, ORDER>((const float*)t.in[k], n, index, chunk);
  else if ((t.dtype[k] & 3) == kBF16)
    v = norm_part<bf16, ORDER>((const bf16*)t.in[k], n, index, chunk);
  else
    v = norm_part<f16, ORDER>((const f16*)t.in[k], n, index, chunk);
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
__device__ __forceinline__ void scale_part(const T* p, O* q, uint32_t n,
                                           uint32_t index, uint32_t chunk, float c) {
  const Part part(n, to_boundary(q), index, chunk);
  if (threadIdx.x < part.head) q[threadIdx.x] = (O)((float)p[threadIdx.x] * c);
  uint32_t i = part.begin;
  for (; part.end - i >= kPass; i += kPass) {
    float v[kUnder][kRun];
#pragma unroll
    for (int k = 0; k < kUnder; ++k)
      load_run<T, kRun>(p + i + (k * kThreads + threadIdx.x) * kRun, v[k]);
#pragma unroll
    for (int k = 0; k < kUnder; ++k) {
#pragma unroll
      for (int j = 0; j < kRun; ++j) v[k][j] *= c;
      store_run<O, kRun>((O*)__builtin_assume_aligned(
                             q + i + (k * kThreads + threadIdx.x) * kRun, 16), v[k]);
    }
  }
  for (i += threadIdx.x * kRun; i < part.end; i += kThreads * kRun) {
    const int some = (int)(part.end - i);
    float v[kRun];
    load_some<T, kRun>(p + i, some, v, 0.f);
#pragma unroll
    for (int j = 0; j < kRun; ++j) v[j] *= c;
    store_some<O, kRun>(q + i, some, v);
  }
}

template <typename T>
__device__ __forceinline__ void scale_to(const T* p, void* q, int dtype, uint32_t n,
                                         uint32_t index, uint32_t chunk, float c) {
  if (dtype == kF32) scale_part<T, float>(p, (float*)q, n, index, chunk, c);
  else if (dtype == kBF16) scale_part<T, bf16>(p, (bf16*)q, n, index, chunk, c);
  else scale_part<T, f16>(p, (f16*)q, n, index, chunk, c);
}

template <bool OUT>
__global__ __launch_bounds__(kThreads) void scale_kernel(Table<OUT> t,
                                                         uint32_t chunk,
                                                         const float* coef) {
  const float c = *coef;
  if (!OUT && c == 1.f) return;
  const int k = find(t, blockIdx.x);
  const uint32_t index = blockIdx.x - t.first[k], n = t.numel[k];
  const int from = t.dtype[k] & 3, to = t.dtype[k] >> 2;
  if constexpr (OUT) {
    if (from == kF32) scale_to((const float*)t.in[k], t.out[k], to, n, index, chunk, c);
    else if (from == kBF16) scale_to((const bf16*)t.in[k], t.out[k], to, n, index, chunk, c);
    else scale_to((const f16*)t.in[k], t.out[k], to, n, index, chunk, c);
  } else {
    void* p = const_cast<void*>(t.in[k]);
    if (from == kF32) scale_part((const float*)p, (float*)p, n, index, chunk, c);
    else if (from == kBF16) scale_part((const bf16*)p, (bf16*)p, n, index, chunk, c);
    else scale_part((const f16*)p, (f16*)p, n, index, chunk, c);
  }
}

constexpr int64_t kPiece = (int64_t)1 << 31;  // elements of an entry, at most

int64_t blocks_of(int64_t numel, int64_t chunk) {
  // a piece's chunks begin at its first boundary, so they may be one fewer
  return (numel + chunk - 1) / chunk;
}

// Fills a table from element `done` of tensor i on; returns the blocks it takes.
template <bool OUT>
uint32_t fill(const GradTensor* g, int count, int64_t chunk, int& i, int64_t& done,
              Table<OUT>& t) {
  static const int size[3] = {4, 2, 2};
  uint32_t blocks = 0;
  t.count = 0;
  while (i < count && t.count < Table<OUT>::most) {
    const int64_t left = g[i].numel - done;
    const int64_t n = left < kPiece ? left : kPiece;
    if (n > 0) {
      const int k = t.count++;
      t.in[k] = (const char*)g[i].in + done * size[g[i].in_dtype];
      if (OUT) t.out[k] = (char*)g[i].out + done * size[g[i].out_dtype];
      t.numel[k] = (uint32_t)n;
      t.dtype[k] = (uint8_t)(g[i].in_dtype | g[i].out_dtype << 2);
      t.first[k] = blocks;
      blocks += (uint32_t)blocks_of(n, chunk);
    }
    done += n;
    if (done >= g[i].numel) ++i, done = 0;
  }
  return blocks;
}

// Nothing is left to add up here: chunks of one pass end together.
template <bool OUT>
void scale_all(const GradTensor* g, int count, const float* coef, hipStream_t stream) {
  Table<OUT> t;
  int64_t done = 0;
  for (int i = 0; i < count;) {
    const uint32_t n = fill<OUT>(g, count, kPass, i, done, t);
    if (n) scale_kernel<OUT><<<n, kThreads, 0, stream>>>(t, kPass, coef);
  }
}

}  // namespace

// Chunks of a pass for small lists, so that many blocks share them (1 M bf16 values
// in 10 tensors take 5.6 us, 6.1 with 16384 elements; 5 M fp32 ones in 50 take 6.2
// us, 7.1 with 4096, which fill no pass), up to 16384 for large ones, so that few
// partial sums are left.
int64_t grad_norm_blocks(const GradTensor* g, int count, int64_t* chunk) {
  int64_t total = 0;
  for (int i = 0; i < count; ++i) total += g[i].numel;
  int64_t c = kPass;
  while (c < 16384 && total / c > 4096) c *= 2;
  *chunk = c;
  int64_t blocks = 0;
  for (int i = 0; i < count; ++i)
    for (int64_t done = 0; done < g[i].numel; done += kPiece)
      blocks += blocks_of(g[i].numel - done < kPiece ? g[i].numel - done : kPiece, c);
  return blocks;
}

void grad_norm(const GradTensor* g, int count, int64_t chunk, int order,
               double* partial, int64_t blocks, float* norm, float* coef,
               float max_norm, float eps, hipStream_t stream) {
  Table<false> t;
  double* at = partial;
  int64_t done = 0;
  for (int i = 0; i < count;) {
    const uint32_t n = fill<false>(g, count, chunk, i, done, t);
    if (!n) continue;
    const uint32_t c = (uint32_t)chunk;
    if (order == 2) norm_kernel<2><<<n, kThreads, 0, stream>>>(t, c, at);
    else if (order == 1) norm_kernel<1><<<n, kThreads, 0, stream>>>(t, c, at);
    else norm_kernel<0><<<n, kThreads, 0, stream>>>(t, c, at);
    at += n;
  }
  if (order == 2)
    norm_join_kernel<2><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
  else if (order == 1)
    norm_join_kernel<1><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
  else
    norm_join_kernel<0><<<1, 1024, 0, stream>>>(partial, blocks, norm, coef, max_norm, eps);
}

void grad_scale(const GradTensor* g, int count, const float* coef,
                hipStream_t stream) {
  bool in_place = true;
  for (int i = 0; i < count; ++i) in_place = in_place && g[i].in == g[i].out;
  if (in_place) scale_all<false>(g, count, coef, stream);
  else scale_all<true>(g, count, coef, stream);
}

}  // namespace blk
