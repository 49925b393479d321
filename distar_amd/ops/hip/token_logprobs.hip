// Log probabilities of given tokens, the entropy of their distributions and
// the likeliest alternatives, from one reading of the logits.
//
//   y_j = (l_j - m) / (T ln 2) over the allowed places, m = max l
//   S = sum 2^y,  U = sum y 2^y
//   logprob = ln 2 (y_t - log2 S)       H = ln 2 (log2 S - U / S)
//   dl_j = (g_lp (d_tj - p_j) - g_H p_j (log p_j + H)) / T
//
// Forward, a thread runs through its part of the row with a maximum of its own
// that its sums follow, four 16-byte runs at a time with the next four under way;
// the threads' maxima and sums are joined at the end, so a row is read once and
// waits once. 64, 256 or 512 threads take a row. Narrow rows without alternatives
// lie in the registers of 8 or 16 threads instead.
//
// The k alternatives: of 64 maxima over disjoint parts of the row (one of each
// lane) the k-th largest is a bound that at least k elements reach, and few more
// do. Only the few threads whose maximum reaches it look at their part again (read
// again where a row is longer than the registers); what reaches it goes to a list
// in LDS, where each counts how many come before it, and the first k write
// themselves out. Only a row with very many equal logits overflows the list: it is
// searched k times instead.
//
// Backward, the gradient's memory is cut into aligned runs of 16 bytes whatever
// the rows' width, and a run that holds the end of a row takes a slower way. The
// gradient is rounded once, to the logits' type.
//
// Memory bounds all but the smallest. 65536 x 513 bf16 with a mask: forward 23 us
// (4.4 TB/s), backward 37 us (4.5 TB/s). 2048 x 24320 bf16: forward with 5
// alternatives 30 us (3.3 TB/s), backward 33 us (6.0 TB/s; much of the logits still
// lies in the cache behind the dies' own). 33 x 24320 fp32 with 20 alternatives:
// 12 us, one block's latency a row; 16 x 327 fp32 with a mask and 5: 5 us.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

// An exponent of 2 whose power is 0 in 32 bits. Where a power is multiplied with its
// exponent, an infinite one is replaced by this, and so is a huge one, which a large
// factor could take out of range: 0 times either is 0.
constexpr float kFar = -256.f;

__device__ __forceinline__ float exp2_(float y) {
  return __builtin_amdgcn_exp2f(y);
}

__device__ __forceinline__ float log2_(float s) {
  return __builtin_amdgcn_logf(s);
}

template <typename T>
using Run = T __attribute__((ext_vector_type(Width<T>::v)));

// maximum, S and U of a part of a row; S is NaN if that holds a NaN, or +inf
// (from inf - inf)
struct Stat {
  float m, s, u;
};

__device__ __forceinline__ bool before(float v, int i, float w, int j) {
  return v > w || (v == w && i < j);
}

// n elements of a row (at least one); -inf behind them and where the mask is 0
template <typename T>
__device__ __forceinline__ Run<T> load_masked(const T* l, const uint8_t* mask,
                                              int n) {
  constexpr int V = Width<T>::v;
  Run<T> v;
  if (n >= V) {
    __builtin_memcpy(&v, l, 16);
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = i < n ? l[i] : (T)-kInf;
  }
  if (mask) {
    uint8_t q[V];
    if (n >= V) {
      __builtin_memcpy(q, mask, V);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) q[i] = i < n ? mask[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = q[i] ? v[i] : (T)-kInf;
  }
  return v;
}

// -inf in the places of v whose byte of q is 0
template <typename T>
__device__ __forceinline__ Run<T> masked(Run<T> v, uint64_t q) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 u = __builtin_bit_cast(u32x4, v);
  const uint32_t half[2] = {(uint32_t)q, (uint32_t)(q >> 32)};
#pragma unroll
  for (int d = 0; d < 4; ++d) {
    if constexpr (sizeof(T) == 4) {
      u[d] = half[0] & (0xffu << 8 * d) ? u[d] : 0xff800000u;
    } else {
      const uint32_t two = half[d >> 1] >> 16 * (d & 1);
      const uint32_t keep = (two & 0xffu ? 0xffffu : 0u) | (two & 0xff00u ? 0xffff0000u : 0u);
      const uint32_t inf = (uint32_t)__builtin_bit_cast(uint16_t, (T)-kInf) * 0x10001u;
      u[d] = (u[d] & keep) | (inf & ~keep);
    }
  }
  return __builtin_bit_cast(Run<T>, u);
}

// Nothing computed from v before this is kept for after it: the compiler would
// hold every element's 32-bit form between the maximum and the sums.
template <typename T>
__device__ __forceinline__ void forget(Run<T>& v) {
  typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
  u32x4 u = __builtin_bit_cast(u32x4, v);
  asm volatile("" : "+v"(u));
  v = __builtin_bit_cast(Run<T>, u);
}

constexpr int kList = 1024;         // alternatives' candidates of a block

// What the waves of a row exchange.
template <int TPR>
struct Shared {
  static constexpr int waves = TPR > 64 ? TPR / 64 : 1;
  static constexpr int list = kList / (TPR > 64 ? 1 : 4);   // of a row or wave
  float most[waves];
  Stat stat[waves];
  float lane_most[TPR > 64 ? waves : 4][64];
  float bound;
  float best_v[waves];
  int best_i[waves];
  int count[TPR > 64 ? 1 : 4];
  struct { float v; int i; } list_of[kList];
};

template <int TPR>
__device__ __forceinline__ void row_sync() {
  if constexpr (TPR > 64) {
    __syncthreads();
  } else {
    // one wave: its LDS accesses are in order, the compiler's must be too
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// What a row's first thread leaves: its results but for the alternatives, and
// what the backward pass needs. `given` is the token's logit, -inf if masked.
__device__ __forceinline__ void leave(const LogProbs& a, int64_t row, Stat st,
                                      int64_t token, float given, float scale) {
  const bool ignored = token == a.ignore_index;
  const bool inside = token >= 0 && token < a.width;
  const bool empty = st.m == -kInf && st.s == 0.f;
  const bool bad = st.s != st.s;
  const float nan = __builtin_nanf("");
  const float log2sum = log2_(st.s);
  const float h = bad ? nan : empty ? 0.f : (log2sum - st.u / st.s) * kLn2;
  a.logprob[row] = ignored ? 0.f
                 : !inside || bad ? nan
                 : given == -kInf ? -kInf
                 : ((given - st.m) * scale - log2sum) * kLn2;
  a.entropy[row] = h;
  if (a.stats) {
    // -1: no gradient of the log probability; -2: one through the sum alone, for a
    // token that is not possible has none of its own
    const int place = ignored || !inside ? -1 : given == -kInf ? -2 : (int)token;
    const float4 keep = {bad ? nan : st.m, log2sum, h, __int_as_float(place)};
    *(float4*)(a.stats + row * 4) = keep;
  }
}

template <typename T>
__device__ __forceinline__ float given_logit(const LogProbs& a, int64_t row,
                                             int64_t token) {
  if (token < 0 || token >= a.width) return -kInf;
  if (a.mask && !a.mask[row * a.mask_stride + token]) return -kInf;
  return (float)((const T*)a.logits)[row * a.stride + token];
}

// Rows of at most TPR * V * NV elements, without alternatives.
template <typename T, int TPR, int NV, bool NARROW>
__global__ __launch_bounds__(256) void logprobs_small_kernel(LogProbs a) {
  constexpr int V = Width<T>::v;
  constexpr int RPB = 256 / TPR;
  const int t = threadIdx.x % TPR;
  const float scale = a.inv_temperature * kLog2e;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows;
       row0 += (int64_t)gridDim.x * RPB) {
    const int64_t mine = row0 + threadIdx.x / TPR;
    const int64_t row = mine < a.rows ? mine : a.rows - 1;
    const T* l = (const T*)a.logits + row * a.stride;
    const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const int64_t token = a.tokens[row];
    Run<T> v[NV];
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const RowRun<T, NARROW> run((j * TPR + t) * V, a.width);
      if constexpr (NARROW) {
        v[j] = (Run<T>)(T)-kInf;
        if (run.any()) v[j] = load_masked<T>(l + run.c, mask ? mask + run.c : nullptr,
                                             a.width - run.c);
      } else {
        __builtin_memcpy(&v[j], l + run.at, 16);
      }
    }
    // asked for behind the row, whose loads it would hold up
    const float given = t == 0 ? given_logit<T>(a, row, token) : 0.f;
    if constexpr (!NARROW) {
      if (mask) {
        uint64_t q[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j)
          __builtin_memcpy(&q[j], mask + RowRun<T>((j * TPR + t) * V, a.width).at, V);
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j] = masked<T>(v[j], q[j]);
      }
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const RowRun<T> run((j * TPR + t) * V, a.width);
        if (run.whole()) continue;
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = run.counts(i) ? v[j][i] : (T)-kInf;
      }
    }
    Stat st = {-kInf, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < NV; ++j)
#pragma unroll
      for (int i = 0; i < V; ++i) st.m = fmaxf(st.m, (float)v[j][i]);
    st.m = lanes_max<TPR>(st.m);
    const float m = st.m == -kInf ? 0.f : st.m;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      if (NV > 1 && j * TPR * V >= a.width) break;    // the same for all
      forget<T>(v[j]);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float y = ((float)v[j][i] - m) * scale, e = exp2_(y);
        st.s += e;
        st.u += e * fmaxf(y, kFar);       // e is 0 there
      }
    }
    st.s = lanes_sum<TPR>(st.s);
    st.u = lanes_sum<TPR>(st.u);
    if (t == 0 && mine < a.rows) leave(a, row, st, token, given, scale);
  }
}

// A thread's runs of a row, TPR runs apart, kBatch of them under way together.
template <typename T, int TPR, bool MASKED, int kBatch>
struct Batch {
  static constexpr int V = Width<T>::v;
  Run<T> v[kBatch];
  uint64_t q[MASKED ? kBatch : 1];

  __device__ __forceinline__ void load(const T* l, const uint8_t* mask, int c0,
                                       int width) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      __builtin_memcpy(&v[j], l + RowRun<T>(c0 + j * TPR * V, width).at, 16);
    if constexpr (MASKED) {
#pragma unroll
      for (int j = 0; j < kBatch; ++j)
        __builtin_memcpy(&q[j], mask + RowRun<T>(c0 + j * TPR * V, width).at, V);
    }
  }

  // -inf in the places that the mask or the row's end take away; first: where the
  // first thread's runs begin
  __device__ __forceinline__ void limit(int first, int width) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      if (TPR == 64 && first + j * TPR * V >= width) break;         // the same for all
      if constexpr (MASKED) v[j] = masked<T>(v[j], q[j]);
      const RowRun<T> run(first + threadIdx.x % TPR * V + j * TPR * V, width);
      if (!run.whole()) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[j][i] = run.counts(i) ? v[j][i] : (T)-kInf;
      }
    }
  }
};

// kBatch < 4: rows of one batch, which leave registers for more waves.
template <typename T, int TPR, bool MASKED, int kBatch>
__global__ __launch_bounds__(TPR > 64 ? TPR : 256,
                             TPR > 256 ? 2 : kBatch < 4 ? (MASKED ? 5 : 6) : MASKED ? 3 : 4)
void logprobs_kernel(LogProbs a) {
  constexpr int V = Width<T>::v;
  constexpr int RPB = TPR > 64 ? 1 : 256 / TPR;
  constexpr int W = Shared<TPR>::waves;
  constexpr int kStep = TPR * V * kBatch;
  constexpr bool kOnce = kBatch < 4;
  __shared__ Shared<TPR> sh;
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 63;
  const int wave = TPR > 64 ? threadIdx.x >> 6 : 0;
  const int slot = TPR > 64 ? 0 : threadIdx.x >> 6;     // the wave's list
  const float scale = a.inv_temperature * kLog2e;
  const int width = a.width;
  const bool narrow = width < V;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows;
       row0 += (int64_t)gridDim.x * RPB) {
    const int64_t mine = row0 + threadIdx.x / TPR;
    const bool some = mine < a.rows;
    const int64_t row = some ? mine : a.rows - 1;
    const T* l = (const T*)a.logits + row * a.stride;
    const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    const int64_t token = a.tokens[row];
    Batch<T, TPR, MASKED, kBatch> now;
    if (!narrow) now.load(l, mask, t * V, width);
    // asked for behind the row's first part, whose loads it would hold up
    const float given = t == 0 ? given_logit<T>(a, row, token) : 0.f;

    Stat st = {-kInf, 0.f, 0.f};
    auto add = [&](const Run<T>& v, float m) {
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float y = ((float)v[i] - m) * scale, e = exp2_(y);
        st.s += e;
        st.u += e * fmaxf(y, kFar);       // e is 0 there
      }
    };
    // the sums go over to a larger maximum; returns what to subtract
    auto raise = [&](float most) {
      const float m = fmaxf(st.m, most);
      const float by = m == -kInf ? 0.f : m;
      const float d = fmaxf((st.m - by) * scale, kFar), f = exp2_(d);
      st.u = (st.u + d * st.s) * f;
      st.s *= f;
      st.m = m;
      return by;
    };
    if (narrow) {
      if (t == 0) {
        const Run<T> v = load_masked<T>(l, mask, width);
        float most = -kInf;
#pragma unroll
        for (int i = 0; i < V; ++i) most = fmaxf(most, (float)v[i]);
        add(v, raise(most));
      }
    } else {
      Batch<T, TPR, MASKED, kBatch> next;
      for (int c = 0; c < width; c += kStep) {
        const bool more = !kOnce && c + kStep < width;
        if (more) next.load(l, mask, c + kStep + t * V, width);
        now.limit(c, width);
        float most = -kInf;
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (TPR == 64 && c + j * TPR * V >= width) break;         // the same for all
#pragma unroll
          for (int i = 0; i < V; ++i) most = fmaxf(most, (float)now.v[j][i]);
        }
        const float m = raise(most);
#pragma unroll
        for (int j = 0; j < kBatch; ++j) {
          if (c + j * TPR * V >= width) break;          // the same for all
          forget<T>(now.v[j]);
          add(now.v[j], m);
        }
        if (kOnce) break;
        if (TPR > 64 || more) now = next;               // a row of one batch stays
      }
    }
    const float most = st.m;              // this thread's maximum
    st.m = lanes_max<64>(most);
    if constexpr (TPR > 64) {
      if (lane == 0) sh.most[wave] = st.m;
      sh.lane_most[wave][lane] = most;
      __syncthreads();
#pragma unroll
      for (int w = 0; w < W; ++w) st.m = fmaxf(st.m, sh.most[w]);
    }
    {
      const float by = st.m == -kInf ? 0.f : st.m;
      const float d = fmaxf((most - by) * scale, kFar), f = exp2_(d);
      st.u = lanes_sum<64>((st.u + d * st.s) * f);
      st.s = lanes_sum<64>(st.s * f);
    }
    if constexpr (TPR > 64) {
      if (lane == 0) sh.stat[wave] = st;
      __syncthreads();
      st.s = st.u = 0.f;
#pragma unroll
      for (int w = 0; w < W; ++w) st.s += sh.stat[w].s, st.u += sh.stat[w].u;
    }
    if (t == 0 && some) leave(a, row, st, token, given, scale);
    if (!a.top_k) {
      if constexpr (TPR > 64) __syncthreads();     // sh is used by the next row
      continue;
    }

    const bool bad = st.s != st.s;
    const bool none = bad || st.m == -kInf || !some;
    const float log2sum = log2_(st.s);
    const int K = a.top_k;
    float* out_lp = a.top_logprobs + row * K;
    int64_t* out_t = a.top_tokens + row * K;
    // the elements of a run, one by one: what follows is rare, so it is small
    // rather than fast (a lone row's time is also that of fetching its code)
    auto each_of = [&](int c, auto f) {
      const Run<T> v = load_masked<T>(l + c, MASKED ? mask + c : nullptr, width - c);
#pragma unroll
      for (int i = 0; i < V; ++i) f((float)v[i], c + i);
    };
    // the K-th largest of 64 lanes' maxima: the largest K times, or the least of
    // those with fewer than K above them (which takes as long as 6 times)
    float bound = most;
    if (TPR == 64 || wave == 0) {
      float g = most;
      if constexpr (TPR > 64)
        for (int w = 1; w < W; ++w) g = fmaxf(g, sh.lane_most[w][lane]);
      if (K <= 6) {
        for (int k = 0; k < K; ++k) {
          bound = lanes_max<64>(g);
          const uint64_t who = __ballot(g == bound);
          if (who && lane == __ffsll((unsigned long long)who) - 1) g = -kInf;
        }
      } else {
        sh.lane_most[slot][lane] = g;
        row_sync<64>();
        int above = 0;
#pragma unroll 2
        for (int o = 0; o < 64; o += 4) {
          const float4 q = *(const float4*)&sh.lane_most[slot][o];
          above += q.x > g;
          above += q.y > g;
          above += q.z > g;
          above += q.w > g;
        }
        bound = -lanes_max<64>(above < K ? -g : -kInf);
      }
      if (lane == 0) {
        sh.count[slot] = 0;
        sh.bound = bound;
      }
    }
    row_sync<TPR>();
    if constexpr (TPR > 64) bound = sh.bound;
    auto* list = sh.list_of + slot * Shared<TPR>::list;
    if (!none && most >= bound)
      for (int c0 = t * V; c0 < width; c0 += kStep) {
        int hit = 1;                      // a narrow row is one run
        if (!narrow) {
          hit = 0;
          if (!kOnce && (TPR > 64 || width > kStep)) {
            now.load(l, mask, c0, width);
            now.limit(c0 - t * V, width);
          }
#pragma unroll
          for (int j = 0; j < kBatch; ++j) {
            if (TPR == 64 && c0 - t * V + j * TPR * V >= width) break;
            float r = -kInf;
#pragma unroll
            for (int i = 0; i < V; ++i) r = fmaxf(r, (float)now.v[j][i]);
            hit |= (r >= bound) << j;
          }
        }
        for (; hit; hit &= hit - 1) {
          const int c = c0 + (__ffs(hit) - 1) * TPR * V;
          if (c >= width) continue;
          each_of(c, [&](float x, int i) {
            if (x >= bound && x > -kInf) {
              const int n = atomicAdd(&sh.count[slot], 1);
              if (n < Shared<TPR>::list) {
                list[n].v = x;
                list[n].i = i;
              }
            }
          });
        }
      }
    row_sync<TPR>();
    const int n = none ? 0 : sh.count[slot];
    if (n <= Shared<TPR>::list) {
      for (int q = t; q < n; q += TPR) {
        const float x = list[q].v;
        const int c = list[q].i;
        int rank = 0;
#pragma unroll 4
        for (int o = 0; o < n; ++o) rank += before(list[o].v, list[o].i, x, c);
        if (rank < K) {
          out_lp[rank] = ((x - st.m) * scale - log2sum) * kLn2;
          out_t[rank] = c;
        }
      }
      if (some)
        for (int k = n + t; k < K; k += TPR) {
          out_lp[k] = bad ? __builtin_nanf("") : -kInf;
          out_t[k] = -1;
        }
    } else {
      // each the best behind the one before it; the list held more than K
      float last_v = kInf;
      int last_i = -1;
      for (int k = 0; k < K; ++k) {
        float bv = -kInf;
        int bi = INT32_MAX;
        for (int c = t * V; c < width; c += TPR * V)
          each_of(c, [&](float x, int i) {
            if (x > -kInf && before(last_v, last_i, x, i) && before(x, i, bv, bi)) {
              bv = x;
              bi = i;
            }
          });
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
          const float ov = __shfl_xor(bv, o, 64);
          const int oi = __shfl_xor(bi, o, 64);
          if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
        }
        if constexpr (TPR > 64) {
          __syncthreads();
          if (lane == 0) sh.best_v[wave] = bv, sh.best_i[wave] = bi;
          __syncthreads();
          bv = sh.best_v[0], bi = sh.best_i[0];
          for (int w = 1; w < W; ++w)
            if (before(sh.best_v[w], sh.best_i[w], bv, bi))
              bv = sh.best_v[w], bi = sh.best_i[w];
        }
        if (t == 0) {
          out_lp[k] = ((bv - st.m) * scale - log2sum) * kLn2;
          out_t[k] = bi;
        }
        last_v = bv, last_i = bi;
      }
    }
    row_sync<TPR>();
  }
}

// n / d for n < 2^31 by a product: m = ceil(2^(31 + s) / d), 2^s >= d
struct Divide {
  uint32_t m, s;
};

Divide divide_by(uint32_t d) {
  uint32_t s = 0;
  while ((1ull << s) < d) ++s;
  return {(uint32_t)(((1ull << (31 + s)) + d - 1) / d), s};
}

__device__ __forceinline__ uint32_t over(uint32_t n, Divide d) {
  return (uint32_t)(((uint64_t)n * d.m) >> (31 + d.s));
}

struct RowGrad {
  float m, log2sum, h, glp, gh;
  int token;
};

__device__ __forceinline__ RowGrad row_grad(const LogProbsBwd& a, int64_t row) {
  const float4 s = *(const float4*)(a.stats + row * 4);
  RowGrad r;
  r.m = s.x, r.log2sum = s.y, r.h = s.z;
  r.token = __float_as_int(s.w);
  r.glp = a.dlogprob && r.token != -1 ? a.dlogprob[row] : 0.f;
  r.gh = a.dentropy ? a.dentropy[row] : 0.f;
  return r;
}

__device__ __forceinline__ float logit_grad(const RowGrad& r, float l, int c,
                                            float scale, float inv_t) {
  const float y = (l - r.m) * scale - r.log2sum;
  const float p = exp2_(y);
  float d = -p * (r.glp + r.gh * (fmaxf(y, kFar) * kLn2 + r.h));
  d = y != y ? y : d;
  d += c == r.token ? r.glp : 0.f;
  return r.m == -kInf ? 0.f : d * inv_t;      // a row without any token
}

constexpr int kBwdRuns = 2;           // runs a thread takes

// FLAT: logits (and mask) without gaps between rows of at least one run, so that
// a run is one load whatever rows it holds.
template <typename T, bool FLAT, bool MASKED>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(LogProbsBwd a,
                                                           Divide by_width) {
  constexpr int V = Width<T>::v;
  const float inv_t = a.inv_temperature, scale = inv_t * kLog2e;
  const int width = a.width;
  const int64_t total = a.rows * width;
  const int64_t base = (int64_t)blockIdx.x * (256 * V * kBwdRuns);
  const int64_t row_b = base / width;
  const uint32_t off_b = (uint32_t)(base - row_b * width);
  if constexpr (FLAT) {
    float d[kBwdRuns][V];
    uint8_t keep[kBwdRuns][V];
    RowGrad r[kBwdRuns];
    int64_t row[kBwdRuns], at[kBwdRuns];
    int c[kBwdRuns];
#pragma unroll
    for (int k = 0; k < kBwdRuns; ++k) {
      // the last run moves back to end with the gradient
      const int64_t o = base + (k * 256 + threadIdx.x) * V;
      at[k] = o < total - V ? o : total - V;
      load_run<T, V>((const T*)a.logits + at[k], d[k]);
      if constexpr (MASKED) __builtin_memcpy(keep[k], a.mask + at[k], V);
      if (at[k] >= base) {
        const uint32_t n = off_b + (uint32_t)(at[k] - base);
        const uint32_t q = over(n, by_width);
        row[k] = row_b + q;
        c[k] = (int)(n - q * (uint32_t)width);
      } else {
        row[k] = at[k] / width;
        c[k] = (int)(at[k] - row[k] * width);
      }
      r[k] = row_grad(a, row[k]);
    }
#pragma unroll
    for (int k = 0; k < kBwdRuns; ++k) {
      const int64_t o = base + (k * 256 + threadIdx.x) * V;
      const int here = width - c[k];      // elements of the first row
      if (here >= V) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          d[k][i] = logit_grad(r[k], d[k][i], c[k] + i, scale, inv_t);
      } else {
        const RowGrad next = row_grad(a, row[k] + 1);
#pragma unroll
        for (int i = 0; i < V; ++i)
          d[k][i] = i < here ? logit_grad(r[k], d[k][i], c[k] + i, scale, inv_t)
                             : logit_grad(next, d[k][i], i - here, scale, inv_t);
      }
      if constexpr (MASKED) {
#pragma unroll
        for (int i = 0; i < V; ++i) d[k][i] = keep[k][i] ? d[k][i] : 0.f;
      }
      if (at[k] == o) {
        store_run<T, V>((T*)a.dlogits + o, d[k]);
      } else if (o < total) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          if (at[k] + i >= o) ((T*)a.dlogits)[at[k] + i] = (T)d[k][i];
      }
    }
  } else {
    for (int k = 0; k < kBwdRuns; ++k) {
      const uint32_t o = (k * 256 + threadIdx.x) * V;
      const int64_t left = total - (base + o);
      if (left <= 0) break;
      const int n = left < V ? (int)left : V;
      const uint32_t q = over(off_b + o, by_width);
      int64_t row = row_b + q;
      int c = (int)(off_b + o - q * (uint32_t)width);
      const T* l = (const T*)a.logits + row * a.stride;
      const uint8_t* mask = a.mask + row * a.mask_stride;
      RowGrad r = row_grad(a, row);
      float d[V];
      if (n == V && c + V <= width) {
        uint8_t keep[V];
        load_run<T, V>(l + c, d);
        if constexpr (MASKED) __builtin_memcpy(keep, mask + c, V);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = logit_grad(r, d[i], c + i, scale, inv_t);
          if constexpr (MASKED) d[i] = keep[i] ? d[i] : 0.f;
        }
        store_run<T, V>((T*)a.dlogits + base + o, d);
      } else {
        for (int i = 0; i < n; ++i) {
          float x = logit_grad(r, (float)l[c], c, scale, inv_t);
          if constexpr (MASKED) x = mask[c] ? x : 0.f;
          ((T*)a.dlogits)[base + o + i] = (T)x;
          if (++c == width && i + 1 < n) {
            c = 0;
            l += a.stride;
            if constexpr (MASKED) mask += a.mask_stride;
            r = row_grad(a, ++row);
          }
        }
      }
    }
  }
}

template <typename T, int TPR, int NV, bool NARROW = false>
void fwd_small(const LogProbs& a, hipStream_t stream) {
  const int64_t need = (a.rows + 256 / TPR - 1) / (256 / TPR);
  const dim3 grid((unsigned)(need < (1 << 20) ? need : (1 << 20)));
  logprobs_small_kernel<T, TPR, NV, NARROW><<<grid, 256, 0, stream>>>(a);
}

template <typename T, int TPR, int kBatch = 4>
void fwd_as(const LogProbs& a, hipStream_t stream) {
  const int64_t rpb = TPR > 64 ? 1 : 256 / TPR;
  const int64_t need = (a.rows + rpb - 1) / rpb;
  const dim3 grid((unsigned)(need < (1 << 20) ? need : (1 << 20)));
  if (a.mask)
    logprobs_kernel<T, TPR, true, kBatch><<<grid, TPR > 64 ? TPR : 256, 0, stream>>>(a);
  else
    logprobs_kernel<T, TPR, false, kBatch><<<grid, TPR > 64 ? TPR : 256, 0, stream>>>(a);
}

// Rows of up to 128 runs lie in registers (65536 x 513 bf16: 16 us, 52 us by a wave
// that runs through the row). 49 to 64 runs share the variant of 80: 65536 x 512 bf16
// takes 15.0 us, 13.9 with a variant of its own, and 21.3 and 20.7 with a mask. Longer
// ones take a wave up to 256 runs (8192 x 2000: 10 us, 47 us with 256 threads; of at
// most 128 runs, with alternatives, by a kernel that holds no second batch: 65536 x
// 513 with a mask and 5 of them 84 us, 148 us by the general one), then 256 threads
// (2048 x 24320: 29 us, 38 us with 512), and 512 where rows are too few to fill the
// chip (33 x 24320 fp32 with 20 alternatives: 12.3 us, 14.6 us with 256).
template <typename T>
void fwd(const LogProbs& a, hipStream_t stream) {
  const int n = (a.width + Width<T>::v - 1) / Width<T>::v;    // runs of 16 bytes
  if (!a.top_k && n <= 128) {
    if (a.width < Width<T>::v) fwd_small<T, 8, 1, true>(a, stream);
    else if (n <= 8) fwd_small<T, 8, 1>(a, stream);
    else if (n <= 16) fwd_small<T, 16, 1>(a, stream);
    else if (n <= 32) fwd_small<T, 16, 2>(a, stream);
    else if (n <= 48) fwd_small<T, 16, 3>(a, stream);
    else if (n <= 80) fwd_small<T, 16, 5>(a, stream);
    else fwd_small<T, 16, 8>(a, stream);
  } else if (n <= 64) {
    fwd_as<T, 64, 1>(a, stream);
  } else if (n <= 128) {
    fwd_as<T, 64, 2>(a, stream);
  } else if (n <= 256) {
    fwd_as<T, 64>(a, stream);
  } else if (n <= 1024 || a.rows >= 512) {
    fwd_as<T, 256>(a, stream);
  } else {
    fwd_as<T, 512>(a, stream);
  }
}

template <typename T>
void bwd(const LogProbsBwd& a, hipStream_t stream) {
  constexpr int64_t chunk = 256 * Width<T>::v * kBwdRuns;
  const dim3 grid((unsigned)((a.rows * a.width + chunk - 1) / chunk));
  const Divide by = divide_by((uint32_t)a.width);
  const bool flat = a.width >= Width<T>::v && (a.stride == a.width || a.rows == 1) &&
                    (!a.mask || a.mask_stride == a.width || a.rows == 1);
  if (flat && a.mask)
    logprobs_bwd_kernel<T, true, true><<<grid, 256, 0, stream>>>(a, by);
  else if (flat)
    logprobs_bwd_kernel<T, true, false><<<grid, 256, 0, stream>>>(a, by);
  else if (a.mask)
    logprobs_bwd_kernel<T, false, true><<<grid, 256, 0, stream>>>(a, by);
  else
    logprobs_bwd_kernel<T, false, false><<<grid, 256, 0, stream>>>(a, by);
}

}  // namespace

void token_logprobs_fwd(const LogProbs& a, int dtype, hipStream_t stream) {
  if (dtype == kF32) fwd<float>(a, stream);
  else if (dtype == kBF16) fwd<bf16>(a, stream);
  else fwd<f16>(a, stream);
}

void token_logprobs_bwd(const LogProbsBwd& a, int dtype, hipStream_t stream) {
  if (dtype == kF32) bwd<float>(a, stream);
  else if (dtype == kBF16) bwd<bf16>(a, stream);
  else bwd<f16>(a, stream);
}

}  // namespace blk
