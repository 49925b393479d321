// Log probabilities of given tokens, the entropy of their distributions and
// the likeliest alternatives, from one reading of the logits.
//
//   x_j = (l_j - m) / T over the allowed places, m = max l
//   S = sum e^x,  U = sum x e^x
//   logprob = x_t - log S       H = log S - U / S
//   dl_j = (g_lp (d_tj - p_j) - g_H p_j (log p_j + H)) / T
//
// A place counts as having no probability where the mask is 0, whatever the
// logit there holds, and where the logit is -inf. S and U are 32-bit sums.
// Alternatives are ranked by the logits themselves, equal ones by their index,
// so the temperature's rounding cannot reorder them.
//
// Forward, a row up to 32768 wide is read once and stays in the registers of
// 8 to 1024 threads, which take its maximum, then the sums, then look for the
// alternatives in it. A wider one runs through 1024 threads, each with a maximum
// of its own that its sums follow, and is read again for alternatives.
//
// The k alternatives: of 64 maxima over disjoint parts of the row (one of each
// lane) the k-th largest is a bound that at least k elements reach, and few more
// do. Those that reach it go to a list in LDS, where each counts how many come
// before it; the first k write themselves out. Only a row with very many equal
// logits overflows the list: it is searched k times instead.
//
// Backward, the gradient's memory is cut into aligned runs of 16 bytes whatever
// the rows' width, and a run that holds the end of a row takes a slower way.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;

__device__ __forceinline__ float exp_(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// maximum, S and U of a part of a row
struct Stat {
  float m, s, u;
};

__device__ __forceinline__ Stat join(Stat a, Stat b, float inv_t) {
  Stat r;
  r.m = fmaxf(a.m, b.m);
  if (r.m == -kInf) return {-kInf, a.s + b.s, 0.f};   // S is 0, or NaN to keep
  const float da = a.m == -kInf ? 0.f : (a.m - r.m) * inv_t;
  const float db = b.m == -kInf ? 0.f : (b.m - r.m) * inv_t;
  const float ea = exp_(da), eb = exp_(db);
  r.s = a.s * ea + b.s * eb;
  r.u = (a.u + da * a.s) * ea + (b.u + db * b.s) * eb;
  return r;
}

__device__ __forceinline__ bool before(float v, int i, float w, int j) {
  return v > w || (v == w && i < j);
}

template <typename T, int V>
__device__ __forceinline__ void load_masked(const T* l, const uint8_t* mask,
                                            int n, float (&v)[V]) {
  load_some<T, V>(l, n, v, -kInf);
  if (mask) {
    uint8_t q[V];
    if (n >= V) {
      __builtin_memcpy(q, mask, V);
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) q[i] = i < n ? mask[i] : 0;
    }
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = q[i] ? v[i] : -kInf;
  }
}

constexpr int kList = 1024;         // alternatives' candidates of a block

// What the waves of a row exchange.
template <int TPR>
struct Shared {
  static constexpr int waves = TPR > 64 ? TPR / 64 : 1;
  static constexpr int rows = TPR > 64 ? 1 : 256 / TPR;
  static constexpr int list = kList / (TPR > 64 ? 1 : 4);   // of a row or wave
  float most[waves];
  Stat stat[waves];
  float lane_most[TPR > 64 ? waves : 1][64];
  float bound;
  float best_v[waves];
  int best_i[waves];
  int count[TPR > 64 ? 1 : 4];
  float list_v[kList];
  int list_i[kList];
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

// A row of at most TPR * V * NV elements in registers (NV > 0), or one of any
// width that is loaded again each time (NV = 0).
template <typename T, int TPR, int NV>
__global__ __launch_bounds__(TPR > 64 ? TPR : 256)
void logprobs_kernel(LogProbs a) {
  constexpr int V = Width<T>::v;
  constexpr int RPB = TPR > 64 ? 1 : 256 / TPR;
  constexpr int R = NV ? NV : 1;
  __shared__ Shared<TPR> sh;
  const int t = threadIdx.x % TPR, lane = threadIdx.x & 63;
  const int wave = TPR > 64 ? threadIdx.x >> 6 : 0;
  const int slot = TPR > 64 ? 0 : threadIdx.x >> 6;     // the wave's list
  const float inv_t = a.inv_temperature;
  for (int64_t row0 = (int64_t)blockIdx.x * RPB; row0 < a.rows;
       row0 += (int64_t)gridDim.x * RPB) {
    const int64_t row = row0 + threadIdx.x / TPR;
    const int width = row < a.rows ? a.width : 0;
    const int64_t at = row < a.rows ? row : 0;
    const T* l = (const T*)a.logits + at * a.stride;
    const uint8_t* mask = a.mask ? a.mask + at * a.mask_stride : nullptr;
    // the given token's logit, asked for before the row
    const int64_t token = a.tokens[at];
    const bool inside = token >= 0 && token < a.width;
    const float given = inside && (!mask || mask[token]) ? (float)l[token] : -kInf;

    float v[R][V];
    float most = -kInf;                 // this thread's maximum
    Stat st = {-kInf, 0.f, 0.f};
    if constexpr (NV > 0) {
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        const int c = (j * TPR + t) * V;
        if (c < width) {
          load_masked<T, V>(l + c, mask ? mask + c : nullptr, width - c, v[j]);
        } else {
#pragma unroll
          for (int i = 0; i < V; ++i) v[j][i] = -kInf;
        }
      }
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int i = 0; i < V; ++i) most = fmaxf(most, v[j][i]);
      st.m = lanes_max<TPR < 64 ? TPR : 64>(most);
      if constexpr (TPR > 64) {
        if (lane == 0) sh.most[wave] = st.m;
        sh.lane_most[wave][lane] = most;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < Shared<TPR>::waves; ++w) st.m = fmaxf(st.m, sh.most[w]);
      }
      const float m = st.m == -kInf ? 0.f : st.m;
#pragma unroll
      for (int j = 0; j < NV; ++j) {
        if (NV > 1 && j * TPR * V >= a.width) break;    // the same for all
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = (v[j][i] - m) * inv_t, e = exp_(x);
          st.s += e;
          st.u += e * fmaxf(x, -1e30f);       // e is 0 there
        }
      }
      st.s = lanes_sum<TPR < 64 ? TPR : 64>(st.s);
      st.u = lanes_sum<TPR < 64 ? TPR : 64>(st.u);
      if constexpr (TPR > 64) {
        if (lane == 0) sh.stat[wave] = st;
        __syncthreads();
        st.s = st.u = 0.f;
#pragma unroll
        for (int w = 0; w < Shared<TPR>::waves; ++w)
          st.s += sh.stat[w].s, st.u += sh.stat[w].u;
      }
    } else {
      for (int c = t * V; c < width; c += TPR * V) {
        load_masked<T, V>(l + c, mask ? mask + c : nullptr, width - c, v[0]);
        Stat q = {v[0][0], 0.f, 0.f};
#pragma unroll
        for (int i = 1; i < V; ++i) q.m = fmaxf(q.m, v[0][i]);
        const float m = q.m == -kInf ? 0.f : q.m;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float x = (v[0][i] - m) * inv_t, e = exp_(x);
          q.s += e;
          q.u += e * fmaxf(x, -1e30f);
        }
        st = join(st, q, inv_t);
      }
      most = st.m;
#pragma unroll
      for (int o = 1; o < 64; o <<= 1)
        st = join(st, {__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64),
                       __shfl_xor(st.u, o, 64)}, inv_t);
      if (lane == 0) sh.stat[wave] = st;
      sh.lane_most[wave][lane] = most;
      __syncthreads();
      st = sh.stat[0];
      for (int w = 1; w < Shared<TPR>::waves; ++w) st = join(st, sh.stat[w], inv_t);
    }
    const bool empty = st.m == -kInf && st.s == 0.f;
    // a NaN, or an infinite logit, leaves no distribution
    const bool bad = !empty && !(st.s > 0.f && st.s < kInf && st.m < kInf);
    const float nan = __builtin_nanf("");
    const float logsum = bad ? nan : __logf(st.s);
    if (t == 0 && width) {
      const bool ignored = token == a.ignore_index;
      const float h = bad ? nan : empty ? 0.f : logsum - st.u / st.s;
      float lp;
      if (ignored) lp = 0.f;
      else if (!inside || bad) lp = nan;
      else if (given == -kInf) lp = -kInf;
      else lp = (given - st.m) * inv_t - logsum;
      a.logprob[row] = lp;
      a.entropy[row] = h;
      if (a.stats) {
        const float4 keep = {bad ? nan : st.m, logsum, h,
                             __int_as_float(ignored ? -1 : inside ? (int)token : -2)};
        *(float4*)(a.stats + row * 4) = keep;
      }
    }
    if (!a.top_k) {
      if constexpr (TPR > 64) __syncthreads();     // sh is used by the next row
      continue;
    }

    if constexpr (TPR >= 64) {
      const int K = a.top_k;
      float* out_lp = a.top_logprobs + row * K;
      int64_t* out_t = a.top_tokens + row * K;
      const bool none = bad || empty;
      auto each = [&](auto f) {
        if constexpr (NV > 0) {
#pragma unroll
          for (int j = 0; j < NV; ++j)
#pragma unroll
            for (int i = 0; i < V; ++i) f(v[j][i], (j * TPR + t) * V + i);
        } else {
          for (int c = t * V; c < width; c += TPR * V) {
            load_masked<T, V>(l + c, mask ? mask + c : nullptr, width - c, v[0]);
#pragma unroll
            for (int i = 0; i < V; ++i) f(v[0][i], c + i);
          }
        }
      };
      // the K-th largest of 64 lanes' maxima
      float bound = most;
      if (TPR == 64 || wave == 0) {
        float g = most;
        if constexpr (TPR > 64)
          for (int w = 1; w < Shared<TPR>::waves; ++w)
            g = fmaxf(g, sh.lane_most[w][lane]);
        for (int k = 0; k < K; ++k) {
          bound = lanes_max<64>(g);
          const uint64_t who = __ballot(g == bound);
          if (who && lane == __ffsll((unsigned long long)who) - 1) g = -kInf;
        }
        if (lane == 0) {
          sh.count[slot] = 0;
          sh.bound = bound;
        }
      }
      row_sync<TPR>();
      if constexpr (TPR > 64) bound = sh.bound;
      const int base = slot * Shared<TPR>::list;
      if (!none && most >= bound)
        each([&](float x, int c) {
          if (x >= bound && x > -kInf) {
            const int n = atomicAdd(&sh.count[slot], 1);
            if (n < Shared<TPR>::list) {
              sh.list_v[base + n] = x;
              sh.list_i[base + n] = c;
            }
          }
        });
      row_sync<TPR>();
      const int n = none ? 0 : sh.count[slot];
      if (n <= Shared<TPR>::list) {
        for (int q = t; q < n; q += TPR) {
          const float x = sh.list_v[base + q];
          const int c = sh.list_i[base + q];
          int rank = 0;
          for (int o = 0; o < n; ++o)
            rank += before(sh.list_v[base + o], sh.list_i[base + o], x, c);
          if (rank < K) {
            out_lp[rank] = (x - st.m) * inv_t - logsum;
            out_t[rank] = c;
          }
        }
        if (width)
          for (int k = n + t; k < K; k += TPR) {
            out_lp[k] = bad ? nan : -kInf;
            out_t[k] = -1;
          }
      } else {
        // each the best behind the one before it
        float last_v = kInf;
        int last_i = -1;
        for (int k = 0; k < K; ++k) {
          float bv = -kInf;
          int bi = INT32_MAX;
          each([&](float x, int c) {
            if (x > -kInf && before(last_v, last_i, x, c) && before(x, c, bv, bi)) {
              bv = x;
              bi = c;
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
            for (int w = 1; w < Shared<TPR>::waves; ++w)
              if (before(sh.best_v[w], sh.best_i[w], bv, bi))
                bv = sh.best_v[w], bi = sh.best_i[w];
          }
          // the list held more than K, so there is one
          if (t == 0) {
            out_lp[k] = (bv - st.m) * inv_t - logsum;
            out_t[k] = bi;
          }
          last_v = bv, last_i = bi;
        }
      }
      row_sync<TPR>();
    }
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
  float m, logsum, h, glp, gh;
  int token;
  bool empty;
};

__device__ __forceinline__ RowGrad row_grad(const LogProbsBwd& a, int64_t row) {
  const float4 s = *(const float4*)(a.stats + row * 4);
  RowGrad r;
  r.m = s.x, r.logsum = s.y, r.h = s.z;
  r.token = __float_as_int(s.w);
  r.glp = a.dlogprob && r.token != -1 ? a.dlogprob[row] : 0.f;
  r.gh = a.dentropy ? a.dentropy[row] : 0.f;
  r.empty = r.m == -kInf;
  return r;
}

__device__ __forceinline__ float logit_grad(const RowGrad& r, float l, int c,
                                            float inv_t) {
  const float lp = (l - r.m) * inv_t - r.logsum;
  const float p = exp_(lp);
  float d = -p * (r.glp + r.gh * (fmaxf(lp, -1e30f) + r.h));
  d = lp != lp ? lp : d;
  d += c == r.token ? r.glp : 0.f;
  return r.empty ? 0.f : d * inv_t;
}

constexpr int kBwdRuns = 4;           // runs a thread takes

template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(LogProbsBwd a,
                                                           Divide by_width) {
  constexpr int V = Width<T>::v;
  const float inv_t = a.inv_temperature;
  const int64_t total = a.rows * a.width;
  const int64_t base = (int64_t)blockIdx.x * (256 * V * kBwdRuns);
  const int64_t row_b = base / a.width;
  const uint32_t off_b = (uint32_t)(base - row_b * a.width);
#pragma unroll
  for (int k = 0; k < kBwdRuns; ++k) {
    const uint32_t o = (k * 256 + threadIdx.x) * V;
    if (base + o >= total) break;
    const uint32_t q = over(off_b + o, by_width);
    int64_t row = row_b + q;
    int c = (int)(off_b + o - q * (uint32_t)a.width);
    T* out = (T*)a.dlogits + base + o;
    float d[V];
    RowGrad r = row_grad(a, row);
    if (c + V <= a.width) {
      load_run<T, V>((const T*)a.logits + row * a.stride + c, d);
      uint8_t allowed[V];
      if (a.mask) __builtin_memcpy(allowed, a.mask + row * a.mask_stride + c, V);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        d[i] = logit_grad(r, d[i], c + i, inv_t);
        if (a.mask && !allowed[i]) d[i] = 0.f;
      }
      store_run<T, V>(out, d);
    } else {
      for (int i = 0; i < V && base + o + i < total; ++i) {
        float x = logit_grad(r, (float)((const T*)a.logits)[row * a.stride + c], c,
                             inv_t);
        if (a.mask && !a.mask[row * a.mask_stride + c]) x = 0.f;
        out[i] = (T)x;
        if (++c == a.width && row + 1 < a.rows) {
          c = 0;
          r = row_grad(a, ++row);
        }
      }
    }
  }
}

template <typename T, int TPR, int NV>
void fwd_as(const LogProbs& a, hipStream_t stream) {
  constexpr int rpb = TPR > 64 ? 1 : 256 / TPR;
  const int64_t need = (a.rows + rpb - 1) / rpb;
  const dim3 grid((unsigned)(need < (1 << 20) ? need : (1 << 20)));
  logprobs_kernel<T, TPR, NV><<<grid, TPR > 64 ? TPR : 256, 0, stream>>>(a);
}

template <typename T>
void fwd(const LogProbs& a, hipStream_t stream) {
  const int n = (a.width + Width<T>::v - 1) / Width<T>::v;    // runs of 16 bytes
  if (n <= 8 && !a.top_k) fwd_as<T, 8, 1>(a, stream);
  else if (n <= 64) fwd_as<T, 64, 1>(a, stream);
  else if (n <= 128) fwd_as<T, 64, 2>(a, stream);
  else if (n <= 256) fwd_as<T, 64, 4>(a, stream);
  else if (n <= 512) fwd_as<T, 256, 2>(a, stream);
  else if (n <= 1024) fwd_as<T, 256, 4>(a, stream);
  else if (n <= 2048) fwd_as<T, 1024, 2>(a, stream);
  else if (n <= 4096) fwd_as<T, 1024, 4>(a, stream);
  else if (sizeof(T) == 4 && n <= 8192) fwd_as<T, 1024, sizeof(T) == 4 ? 8 : 4>(a, stream);
  else fwd_as<T, 1024, 0>(a, stream);
}

template <typename T>
void bwd(const LogProbsBwd& a, hipStream_t stream) {
  constexpr int64_t chunk = 256 * Width<T>::v * kBwdRuns;
  const int64_t blocks = (a.rows * a.width + chunk - 1) / chunk;
  logprobs_bwd_kernel<T><<<dim3((unsigned)blocks), 256, 0, stream>>>(
      a, divide_by((uint32_t)a.width));
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
