// Log probabilities of given tokens, the entropy of their distributions and
// the likeliest alternatives, from one reading of the logits.
//
//   x_j = (l_j - m) / T over the allowed places, m = max l
//   S = sum e^x,  U = sum x e^x
//   logprob = x_t - log S       H = log S - U / S
//   dl_j = (g_lp (d_tj - p_j) - g_H p_j (log p_j + H)) / T
//
// A place counts as having no probability where the mask is 0, whatever the
// logit there holds, and where the logit is -inf. m, S and U run along the row
// (S and U are rescaled when m grows), in 32 bits. Alternatives are ranked by
// the logits themselves, equal ones by their index, so the temperature's
// rounding cannot reorder them.
#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr float kInf = __builtin_inff();
constexpr float kLog2e = 1.4426950408889634f;
constexpr int64_t kNone = INT64_MAX;

__device__ __forceinline__ float exp_(float x) {
  return __builtin_amdgcn_exp2f(x * kLog2e);
}

// m, S, U of a part of a row
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

template <typename T, int V>
__device__ __forceinline__ void load_masked(const LogProbs& a, const T* l,
                                            const uint8_t* mask, int c,
                                            float (&v)[V]) {
  const int n = a.width - c;
  load_some<T, V>(l + c, n, v, -kInf);
  if (mask) {
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (i < n && !mask[c + i]) v[i] = -kInf;
  }
}

__device__ __forceinline__ bool before(float v, int i, float w, int j) {
  return v > w || (v == w && i < j);
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_kernel(LogProbs a) {
  constexpr int V = Width<T>::v;
  __shared__ Stat stats[4];
  __shared__ float best_v[4];
  __shared__ int best_i[4];
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const float inv_t = a.inv_temperature;
  for (int64_t row = blockIdx.x; row < a.rows; row += gridDim.x) {
    const T* l = (const T*)a.logits + row * a.stride;
    const uint8_t* mask = a.mask ? a.mask + row * a.mask_stride : nullptr;
    Stat st = {-kInf, 0.f, 0.f};
    for (int c = threadIdx.x * V; c < a.width; c += 256 * V) {
      float v[V];
      load_masked<T, V>(a, l, mask, c, v);
      Stat q = {v[0], 0.f, 0.f};
#pragma unroll
      for (int i = 1; i < V; ++i) q.m = fmaxf(q.m, v[i]);
      const float m = q.m == -kInf ? 0.f : q.m;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float x = (v[i] - m) * inv_t, e = exp_(x);
        q.s += e;
        q.u += e * fmaxf(x, -1e30f);       // e is 0 there
      }
      st = join(st, q, inv_t);
    }
#pragma unroll
    for (int o = 1; o < 64; o <<= 1)
      st = join(st, {__shfl_xor(st.m, o, 64), __shfl_xor(st.s, o, 64),
                     __shfl_xor(st.u, o, 64)}, inv_t);
    __syncthreads();
    if (lane == 0) stats[wave] = st;
    __syncthreads();
    st = stats[0];
    for (int w = 1; w < 4; ++w) st = join(st, stats[w], inv_t);
    const bool empty = st.m == -kInf && st.s == 0.f;
    // a NaN, or an infinite logit, leaves no distribution
    const bool bad = !empty && !(st.s > 0.f && st.s < kInf && st.m < kInf);
    const float nan = __builtin_nanf("");
    const float logsum = bad ? nan : __logf(st.s);
    if (threadIdx.x == 0) {
      const int64_t t = a.tokens[row];
      float lp;
      if (t == a.ignore_index) lp = 0.f;
      else if (t < 0 || t >= a.width || bad) lp = nan;
      else if (empty || (mask && !mask[t])) lp = -kInf;
      else lp = ((float)l[t] - st.m) * inv_t - logsum;
      a.logprob[row] = lp;
      a.entropy[row] = bad ? nan : empty ? 0.f : logsum - st.u / st.s;
      if (a.row_max) {
        a.row_max[row] = bad ? nan : st.m;
        a.row_logsum[row] = logsum;
      }
    }
    // alternatives, each the best behind the one before it
    float last_v = kInf;
    int last_i = -1;
    for (int k = 0; k < a.top_k; ++k) {
      float bv = -kInf;
      int bi = INT32_MAX;
      if (!bad && !empty)
        for (int c = threadIdx.x * V; c < a.width; c += 256 * V) {
          float v[V];
          load_masked<T, V>(a, l, mask, c, v);
#pragma unroll
          for (int i = 0; i < V; ++i)
            if (v[i] > -kInf && before(last_v, last_i, v[i], c + i) &&
                before(v[i], c + i, bv, bi)) {
              bv = v[i];
              bi = c + i;
            }
        }
#pragma unroll
      for (int o = 1; o < 64; o <<= 1) {
        const float ov = __shfl_xor(bv, o, 64);
        const int oi = __shfl_xor(bi, o, 64);
        if (before(ov, oi, bv, bi)) bv = ov, bi = oi;
      }
      __syncthreads();
      if (lane == 0) best_v[wave] = bv, best_i[wave] = bi;
      __syncthreads();
      bv = best_v[0], bi = best_i[0];
      for (int w = 1; w < 4; ++w)
        if (before(best_v[w], best_i[w], bv, bi)) bv = best_v[w], bi = best_i[w];
      if (threadIdx.x == 0) {
        const bool found = bi != INT32_MAX;
        a.top_logprobs[row * a.top_k + k] =
            bad ? nan : found ? (bv - st.m) * inv_t - logsum : -kInf;
        a.top_tokens[row * a.top_k + k] = found ? bi : -1;
      }
      if (bi != INT32_MAX) last_v = bv, last_i = bi;
      else last_v = -kInf;                  // nothing comes behind it
    }
  }
}

template <typename T>
__global__ __launch_bounds__(256) void logprobs_bwd_kernel(LogProbsBwd a) {
  constexpr int V = Width<T>::v;
  const float inv_t = a.inv_temperature;
  for (int64_t row = blockIdx.y; row < a.rows; row += gridDim.y) {
    const int c = (blockIdx.x * 256 + threadIdx.x) * V;
    const int n = a.width - c;
    if (n <= 0) continue;
    const int64_t t = a.tokens[row];
    const float m = a.row_max[row], logsum = a.row_logsum[row];
    const float h = a.entropy[row];
    const float glp = a.dlogprob && t != a.ignore_index ? a.dlogprob[row] : 0.f;
    const float gh = a.dentropy ? a.dentropy[row] : 0.f;
    const bool empty = m == -kInf;
    float v[V];
    load_some<T, V>((const T*)a.logits + row * a.stride + c, n, v, 0.f);
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const bool out = i >= n || empty ||
                       (a.mask && !a.mask[row * a.mask_stride + c + i]);
      const float lp = (v[i] - m) * inv_t - logsum;
      const float p = exp_(lp);
      float d = -p * (glp + gh * (fmaxf(lp, -1e30f) + h));
      if (lp != lp) d = lp;
      if (c + i == t) d += glp;
      v[i] = out ? 0.f : d * inv_t;
    }
    store_some<T, V>((T*)a.dlogits + row * a.width + c, n, v);
  }
}

template <typename T>
void fwd(const LogProbs& a, hipStream_t stream) {
  logprobs_kernel<T><<<dim3((unsigned)(a.rows < 65536 ? a.rows : 65536)), 256,
                       0, stream>>>(a);
}

template <typename T>
void bwd(const LogProbsBwd& a, hipStream_t stream) {
  constexpr int chunk = 256 * Width<T>::v;
  const dim3 grid((a.width + chunk - 1) / chunk,
                  (unsigned)(a.rows < 65535 ? a.rows : 65535));
  logprobs_bwd_kernel<T><<<grid, 256, 0, stream>>>(a);
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
