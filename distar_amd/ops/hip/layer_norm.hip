// Layer normalisation of rows, with the residual sum in front of it.
//
//   s = x + r (stored in x's type: the residual stream)      mu = mean(s)
//   y = (s - mu) rstd w + b            rstd = 1 / sqrt(mean((s - mu)^2) + eps)
//
//   g = dy w,  xhat = (s - mu) rstd
//   ds = rstd (g - mean(g) - xhat mean(g xhat)) + (ds given)
//   dw = sum over rows of dy xhat,  db = sum over rows of dy
//
// Memory bounds both directions: a row is read once into registers, its mean
// and then its variance are taken there (two sums, so that a large mean costs
// no digits), and it is written once. TPR threads hold a row as NV runs of 16
// bytes each; narrow rows share a wave, wide ones take a block. Statistics and
// sums are 32-bit whatever the type. The sum s is rounded to x's type before its
// statistics: it is the stream that the next layers read, and y is its norm.
//
// Backward, a thread keeps the same columns for all rows that its block takes
// and adds dw and db up in registers; a block writes one pair of partial rows,
// and a second kernel adds those up in a fixed order, so equal inputs give
// equal gradients.
//
// 262144 x 256 bf16 with a residual: forward 94 us, 5.7 TB/s over x, r, s and y;
// backward 110 us, 4.9 TB/s over dy, ds, s and dx, and 5 us for the sums of 1024
// blocks (a large copy reaches 4.7 TB/s). 4095 x 1536 fp32: 11 us, and 17 + 4. 16 x 256
// bf16: 2.6 us, a launch.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr int kThreads = 256;

template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* lds) {
  if constexpr (TPR <= 64) {
    return lanes_sum<TPR>(v);
  } else {
    v = lanes_sum<64>(v);
    __syncthreads();                  // the previous sum has been read
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    float t = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 64; ++i) t += lds[i];
    return t;
  }
}

template <typename T, typename WT, int TPR, int NV, bool NARROW>
__global__ __launch_bounds__(TPR > kThreads ? TPR : kThreads)
void ln_fwd_kernel(LayerNormFwd a) {
  constexpr int V = Width<T>::v;
  constexpr int RPB = (TPR > kThreads ? TPR : kThreads) / TPR;
  using Run = RowRun<T, NARROW>;
  __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
  const int t = threadIdx.x % TPR;
  const float inv = 1.f / (float)a.width;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows;
       row0 += (int64_t)gridDim.x * RPB) {
    const int64_t mine = row0 + threadIdx.x / TPR;
    const bool some = mine < a.rows;
    const int64_t row = some ? mine : a.rows - 1;
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* r = (const T*)a.residual + row * a.r_stride;
    float v[NV][V], q[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) Run((j * TPR + t) * V, a.width).load(x, v[j]);
    if (a.residual) {
#pragma unroll
      for (int j = 0; j < NV; ++j) Run((j * TPR + t) * V, a.width).load(r, q[j]);
    }
    float w[NV][V], b[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Run run((j * TPR + t) * V, a.width);
#pragma unroll
      for (int i = 0; i < V; ++i) w[j][i] = 1.f, b[j][i] = 0.f;
      if (a.weight) run.load((const WT*)a.weight, w[j]);
      if (a.bias) run.load((const WT*)a.bias, b[j]);
    }
    if (a.residual) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = rounded<T>(v[j][i] + q[j][i]);
        if (some)
          Run((j * TPR + t) * V, a.width).store((T*)a.s + row * a.width, v[j]);
      }
    }
    float sum = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Run run((j * TPR + t) * V, a.width);
      if (run.whole()) {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += v[j][i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) sum += run.counts(i) ? v[j][i] : 0.f;
      }
    }
    const float mean = row_sum<TPR>(sum, lds) * inv;
    float sq = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Run run((j * TPR + t) * V, a.width);
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] -= mean;
      if (run.whole()) {
#pragma unroll
        for (int i = 0; i < V; ++i) sq += v[j][i] * v[j][i];
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) sq += run.counts(i) ? v[j][i] * v[j][i] : 0.f;
      }
    }
    const float rstd = 1.f / sqrtf(row_sum<TPR>(sq, lds) * inv + a.eps);
    if (!some) continue;                 // only rows that share a block
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[j][i] = v[j][i] * rstd * w[j][i] + b[j][i];
      Run((j * TPR + t) * V, a.width).store((T*)a.y + row * a.width, v[j]);
    }
    if (a.mean && t == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

// Rows too wide for registers: the row is read three times.
template <typename T, typename WT>
__global__ __launch_bounds__(1024) void ln_fwd_wide_kernel(LayerNormFwd a) {
  constexpr int V = Width<T>::v;
  __shared__ float lds[16];
  const float inv = 1.f / (float)a.width;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* x = (const T*)a.x + row * a.x_stride;
    const T* r = (const T*)a.residual + row * a.r_stride;
    T* s = (T*)a.s + row * a.width;
    float v[V], sum = 0.f;
    for (int c = threadIdx.x * V; c < a.width; c += 1024 * V) {
      load_some<T, V>(x + c, a.width - c, v, 0.f);
      if (a.residual) {
        float q[V];
        load_some<T, V>(r + c, a.width - c, q, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = rounded<T>(v[i] + q[i]);
        store_some<T, V>(s + c, a.width - c, v);
      }
#pragma unroll
      for (int i = 0; i < V; ++i) sum += v[i];
    }
    // a thread reads back only what it wrote itself
    const T* in = a.residual ? s : x;
    const float mean = row_sum<1024>(sum, lds) * inv;
    float sq = 0.f;
    for (int c = threadIdx.x * V; c < a.width; c += 1024 * V) {
      load_some<T, V>(in + c, a.width - c, v, mean);
#pragma unroll
      for (int i = 0; i < V; ++i) sq += (v[i] - mean) * (v[i] - mean);
    }
    const float rstd = 1.f / sqrtf(row_sum<1024>(sq, lds) * inv + a.eps);
    for (int c = threadIdx.x * V; c < a.width; c += 1024 * V) {
      float w[V], b[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = 1.f, b[i] = 0.f;
      load_some<T, V>(in + c, a.width - c, v, 0.f);
      if (a.weight) load_some<WT, V>((const WT*)a.weight + c, a.width - c, w, 0.f);
      if (a.bias) load_some<WT, V>((const WT*)a.bias + c, a.width - c, b, 0.f);
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = (v[i] - mean) * rstd * w[i] + b[i];
      store_some<T, V>((T*)a.y + row * a.width + c, a.width - c, w);
    }
    if (a.mean && threadIdx.x == 0) {
      a.mean[row] = mean;
      a.rstd[row] = rstd;
    }
  }
}

template <typename T, typename WT, int TPR, int NV, bool NARROW>
__global__ __launch_bounds__(TPR > kThreads ? TPR : kThreads)
void ln_bwd_kernel(LayerNormBwd a) {
  constexpr int V = Width<T>::v;
  constexpr int NT = TPR > kThreads ? TPR : kThreads;
  constexpr int RPB = NT / TPR;
  using Run = RowRun<T, NARROW>;
  __shared__ float lds[TPR > 64 ? TPR / 64 : 1];
  __shared__ float part[RPB > 1 ? NT * V : 1];
  const int t = threadIdx.x % TPR;
  const float inv = 1.f / (float)a.width;
  float dw[NV][V] = {}, db[NV][V] = {};
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows;
       row0 += (int64_t)gridDim.x * RPB) {
    const int64_t mine = row0 + threadIdx.x / TPR;
    const bool some = mine < a.rows;
    const int64_t row = some ? mine : a.rows - 1;
    float g[NV][V], h[NV][V], o[NV][V];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Run run((j * TPR + t) * V, a.width);
      run.load((const T*)a.dy + row * a.dy_stride, g[j]);
      run.load((const T*)a.s + row * a.s_stride, h[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] = 0.f;
      if (a.ds) run.load((const T*)a.ds + row * a.ds_stride, o[j]);
    }
    const float mean = a.mean[row], rstd = a.rstd[row];
    float s1 = 0.f, s2 = 0.f;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const Run run((j * TPR + t) * V, a.width);
      float w[V];
#pragma unroll
      for (int i = 0; i < V; ++i) w[i] = 1.f;
      if (a.weight) run.load((const WT*)a.weight, w);
      const bool all = run.whole() && some;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        h[j][i] = (h[j][i] - mean) * rstd;
        const float d = all || (some && run.counts(i)) ? g[j][i] : 0.f;
        dw[j][i] += d * h[j][i];
        db[j][i] += d;
        g[j][i] *= w[i];
        s1 += d * w[i];
        s2 += d * w[i] * h[j][i];
      }
    }
    s1 = row_sum<TPR>(s1, lds) * inv;
    s2 = row_sum<TPR>(s2, lds) * inv;
    if (!some) continue;                 // only rows that share a block
#pragma unroll
    for (int j = 0; j < NV; ++j) {
#pragma unroll
      for (int i = 0; i < V; ++i) o[j][i] += rstd * (g[j][i] - s1 - h[j][i] * s2);
      Run((j * TPR + t) * V, a.width).store((T*)a.dx + row * a.width, o[j]);
    }
  }
  if (!a.partial) return;
  // rows that share a block: their sums are added in the order of the groups
#pragma unroll
  for (int j = 0; j < NV; ++j) {
    const Run run((j * TPR + t) * V, a.width);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
      float(&acc)[NV][V] = q ? db : dw;
      if constexpr (RPB > 1) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < V; ++i) part[threadIdx.x * V + i] = acc[j][i];
        __syncthreads();
        if (threadIdx.x < TPR)
          for (int k = 1; k < RPB; ++k)
#pragma unroll
            for (int i = 0; i < V; ++i) acc[j][i] += part[(k * TPR + t) * V + i];
      }
      if (threadIdx.x < TPR)
        run.store(a.partial + ((int64_t)blockIdx.x * 2 + q) * a.width, acc[j]);
    }
  }
}

// Rows too wide for registers: ds here, dw and db by ln_columns_kernel.
template <typename T, typename WT>
__global__ __launch_bounds__(1024) void ln_bwd_wide_kernel(LayerNormBwd a) {
  constexpr int V = Width<T>::v;
  __shared__ float lds[16];
  const float inv = 1.f / (float)a.width;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* dy = (const T*)a.dy + row * a.dy_stride;
    const T* s = (const T*)a.s + row * a.s_stride;
    const float mean = a.mean[row], rstd = a.rstd[row];
    float g[V], h[V], w[V], s1 = 0.f, s2 = 0.f;
    for (int pass = 0; pass < 2; ++pass) {
      for (int c = threadIdx.x * V; c < a.width; c += 1024 * V) {
        const int n = a.width - c;
#pragma unroll
        for (int i = 0; i < V; ++i) w[i] = 1.f;
        load_some<T, V>(dy + c, n, g, 0.f);
        load_some<T, V>(s + c, n, h, mean);
        if (a.weight) load_some<WT, V>((const WT*)a.weight + c, n, w, 0.f);
        float o[V];
#pragma unroll
        for (int i = 0; i < V; ++i) o[i] = 0.f;
        if (pass && a.ds)
          load_some<T, V>((const T*)a.ds + row * a.ds_stride + c, n, o, 0.f);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          g[i] *= w[i];
          h[i] = (h[i] - mean) * rstd;
          if (pass) {
            o[i] += rstd * (g[i] - s1 - h[i] * s2);
          } else {
            s1 += g[i];
            s2 += g[i] * h[i];
          }
        }
        if (pass) store_some<T, V>((T*)a.dx + row * a.width + c, n, o);
      }
      if (!pass) {
        s1 = row_sum<1024>(s1, lds) * inv;
        s2 = row_sum<1024>(s2, lds) * inv;
      }
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void ln_columns_kernel(LayerNormBwd a) {
  const int c = blockIdx.x * 256 + threadIdx.x;
  if (c >= a.width) return;
  float dw = 0.f, db = 0.f;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const float g = (float)((const T*)a.dy)[row * a.dy_stride + c];
    const float s = (float)((const T*)a.s)[row * a.s_stride + c];
    dw += g * ((s - a.mean[row]) * a.rstd[row]);
    db += g;
  }
  a.partial[((int64_t)blockIdx.y * 2 + 0) * a.width + c] = dw;
  a.partial[((int64_t)blockIdx.y * 2 + 1) * a.width + c] = db;
}

// [blocks][2][width] -> dw, db: 16 columns a block, 64 groups of partial rows
// side by side, so that the sum over some thousand blocks is short.
template <typename WT>
__global__ __launch_bounds__(1024) void ln_join_kernel(LayerNormBwd a) {
  __shared__ float lds[64][17];
  const int lane = threadIdx.x % 16, group = threadIdx.x / 16;
  const int64_t cols = 2 * (int64_t)a.width;
  for (int64_t c0 = (int64_t)blockIdx.x * 16; c0 < cols; c0 += (int64_t)gridDim.x * 16) {
    const int64_t c = c0 + lane;
    float v = 0.f;
    if (c < cols)
#pragma unroll 4
      for (int k = group; k < a.blocks; k += 64) v += a.partial[k * cols + c];
    lds[group][lane] = v;
    __syncthreads();
    if (group == 0 && c < cols) {
      for (int k = 1; k < 64; ++k) v += lds[k][lane];
      if (c < a.width)
        ((WT*)a.dweight)[c] = (WT)v;
      else
        ((WT*)a.dbias)[c - a.width] = (WT)v;
    }
    __syncthreads();
  }
}

template <typename T> int runs(int width) {
  return (width + Width<T>::v - 1) / Width<T>::v;
}

// A row's threads are the fewest that hold it in one or two runs each, so that
// narrow rows share a wave and its sums stay within it: 262144 x 256 bf16 takes 43
// us with 32 threads a row, 71 us with 64; 60000 x 1000 39 us with 64 threads of two
// runs, 64 us with 256 of one.

// Rows a pass of a block takes, by the number of 16-byte runs in a row.
int rows_a_block(int n) { return n <= 8 ? 32 : n <= 32 ? 8 : n <= 128 ? 4 : 1; }

constexpr int kMaxRuns = 2048;
constexpr int kWideBlocks = 64;     // row groups of the wide rows' column sums

template <typename T, typename WT>
void fwd(const LayerNormFwd& a, hipStream_t stream) {
  const int n = runs<T>(a.width);
  const int64_t rpb = rows_a_block(n);
  const int64_t need = (a.rows + rpb - 1) / rpb;
  const dim3 grid((unsigned)(need < (1 << 20) ? need : (1 << 20)));
  if (a.width < Width<T>::v)
    ln_fwd_kernel<T, WT, 8, 1, true><<<grid, 256, 0, stream>>>(a);
  else if (n <= 8)
    ln_fwd_kernel<T, WT, 8, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 32)
    ln_fwd_kernel<T, WT, 32, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 64)
    ln_fwd_kernel<T, WT, 64, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 128)
    ln_fwd_kernel<T, WT, 64, 2, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 256)
    ln_fwd_kernel<T, WT, 256, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 512)
    ln_fwd_kernel<T, WT, 256, 2, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 1024)
    ln_fwd_kernel<T, WT, 512, 2, false><<<grid, 512, 0, stream>>>(a);
  else if (n <= kMaxRuns)
    ln_fwd_kernel<T, WT, 1024, 2, false><<<grid, 1024, 0, stream>>>(a);
  else
    ln_fwd_wide_kernel<T, WT><<<grid, 1024, 0, stream>>>(a);
}

template <typename T, typename WT>
void bwd(const LayerNormBwd& a, hipStream_t stream) {
  const int n = runs<T>(a.width);
  const dim3 grid(a.blocks);
  if (a.width < Width<T>::v)
    ln_bwd_kernel<T, WT, 8, 1, true><<<grid, 256, 0, stream>>>(a);
  else if (n <= 8)
    ln_bwd_kernel<T, WT, 8, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 32)
    ln_bwd_kernel<T, WT, 32, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 64)
    ln_bwd_kernel<T, WT, 64, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 128)
    ln_bwd_kernel<T, WT, 64, 2, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 256)
    ln_bwd_kernel<T, WT, 256, 1, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 512)
    ln_bwd_kernel<T, WT, 256, 2, false><<<grid, 256, 0, stream>>>(a);
  else if (n <= 1024)
    ln_bwd_kernel<T, WT, 512, 2, false><<<grid, 512, 0, stream>>>(a);
  else if (n <= kMaxRuns)
    ln_bwd_kernel<T, WT, 1024, 2, false><<<grid, 1024, 0, stream>>>(a);
  else {
    const dim3 rows((unsigned)(a.rows < 65536 ? a.rows : 65536));
    ln_bwd_wide_kernel<T, WT><<<rows, 1024, 0, stream>>>(a);
    if (a.partial)
      ln_columns_kernel<T><<<dim3((a.width + 255) / 256, a.blocks), 256, 0,
                             stream>>>(a);
  }
  if (a.partial) {
    const int64_t need = (2 * (int64_t)a.width + 15) / 16;
    const dim3 columns((unsigned)(need < (1 << 20) ? need : (1 << 20)));   // 2^30 threads
    ln_join_kernel<WT><<<columns, 1024, 0, stream>>>(a);
  }
}

}  // namespace

int layer_norm_bwd_blocks(int64_t rows, int width, int dtype) {
  const int n = dtype == kF32 ? runs<float>(width) : runs<bf16>(width);
  if (n > kMaxRuns) return rows < kWideBlocks ? (int)rows : kWideBlocks;
  const int64_t rpb = rows_a_block(n);
  const int64_t need = (rows + rpb - 1) / rpb;
  // Four blocks a compute unit where a thread has one run of a row, two, with half as
  // many partial rows, where it has two: 60000 x 1000 bf16 takes 73 us, 85 with four
  // (111 with one), 8192 x 4096 bf16 49 and 57; one run, 20000 x 2000, 69 and 57.
  const int64_t most = n > 256 || (n > 64 && n <= 128) ? 512 : 1024;
  return (int)(need < most ? need : most);
}

void layer_norm_fwd(const LayerNormFwd& a, int dtype, int wdtype,
                    hipStream_t stream) {
  if (dtype == kF32) fwd<float, float>(a, stream);
  else if (dtype == kBF16 && wdtype == kF32) fwd<bf16, float>(a, stream);
  else if (dtype == kBF16) fwd<bf16, bf16>(a, stream);
  else if (wdtype == kF32) fwd<f16, float>(a, stream);
  else fwd<f16, f16>(a, stream);
}

void layer_norm_bwd(const LayerNormBwd& a, int dtype, int wdtype,
                    hipStream_t stream) {
  if (dtype == kF32) bwd<float, float>(a, stream);
  else if (dtype == kBF16 && wdtype == kF32) bwd<bf16, float>(a, stream);
  else if (dtype == kBF16) bwd<bf16, bf16>(a, stream);
  else if (wdtype == kF32) bwd<f16, float>(a, stream);
  else bwd<f16, f16>(a, stream);
}

}  // namespace blk
