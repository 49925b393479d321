// Linear layers with their epilogue, and the products of their gradients.
//
//   z = x W^T + b,   y = act(z) + residual
//   dz = dy act'(z), dx = dz W,  dW = dz^T x,  db = sum over rows of dz
//
// One kernel does the three products out[i][j] = sum_r P[i][r] Q[j][r] on the
// matrix cores (16x16x32, 32-bit sums): an operand's r is contiguous in
// memory, or its other index is (W for dx, both operands for dW). Tiles of 32 r
// go through LDS as they lie in memory, in 16-byte chunks whose place in their
// row is XORed with bits of the row, so that the reads of a wave spread over all
// banks; an operand with r across its rows is turned by the transposing LDS
// read. What lies beyond r's end is loaded as zero on both sides, what lies
// beyond i or j is loaded from a valid place and not stored.
//
// y is computed from the 32-bit z and rounded once. z is kept for the backward pass
// in 32 bits too where a slope is taken from it: in the operands' type its rounding
// would weigh as much in the gradients as that of dz, and an fp16 z could overflow
// under a finite y. A relu needs its sign alone and keeps it in the operands' type.
// dz is rounded to that type, because both products take no wider one.
//
// The matrix cores bound long r, memory the rest. 16384 x 4096 by 2048 fp16 with
// gelu, residual and z kept, within a pass: 337 us, 817 TFLOP/s (on its own 309 us, and
// 248 us, 1110 TFLOP/s, without an epilogue: 256 x 256 tiles fill a compute unit, so
// nothing hides their 268 MB); dz 45 us, 5.9 TB/s, dx 292 us (942), dW 244 us (1126)
// and 14 us to join its two parts. 32768 x 997 by 256 bf16 with relu: 39 us, dz and db
// 11 + 4, dx 35, dW 34 + 7.
#include <type_traits>

#include "block_common.h"
#include "block_ops.h"

namespace blk {
namespace {

constexpr int kR = 32;            // r a tile, straight into LDS
constexpr int kSR = 64;           // r a tile, by way of registers

typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef f16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef __attribute__((address_space(3))) s16x4* lds_s16x4;

__device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c, bf16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(
      __builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mma(s16x8 a, s16x8 b, f32x4 c, f16) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(
      __builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

// ---- epilogue

// The normal distribution's cdf; e becomes exp(-z^2 / 2). erfc(x) = exp(-x^2) times a
// polynomial of degree 7 in t = 1 / (1 + 0.36 x) for x >= 0: the form of 7.1.26 in
// Abramowitz and Stegun's handbook, with two more terms, and coefficients of a linear
// program for the least error of the tail, relative to the smaller of 4e-8 and 1e-5 of it.
// The fit is off by at most 1.7e-8, and by 4.2e-6 of the tail, to which 32 bits add some
// 1e-7 and z^2 / 2 roundings of the exponent: far below zero, where z times the tail is
// the output, that is a two-hundredth of bf16's half step and a fortieth of fp16's (the
// handbook's coefficients, within 1.5e-7, are off by 0.2% of the tail at -5 and by 1% at -8).
__device__ __forceinline__ float normal_cdf(float z, float& e) {
  const float x = fabsf(z) * 0.70710678f;
  e = __builtin_amdgcn_exp2f(z * z * -0.72134752f);
  const float t = __builtin_amdgcn_rcpf(fmaf(0.36f, x, 1.f));
  float s = fmaf(-0.163245942f, t, 0.562581674f);
  s = fmaf(s, t, -0.353013857f);
  s = fmaf(s, t, 0.426510795f);
  s = fmaf(s, t, 0.108527269f);
  s = fmaf(s, t, 0.216420075f);
  s = fmaf(s, t, 0.202220012f);
  const float tail = 0.5f * s * t * e;
  return z < 0.f ? tail : 1.f - tail;
}

template <int ACT>
__device__ __forceinline__ float act(float z) {
  if constexpr (ACT == kRelu) return z < 0.f ? 0.f : z;       // keeps a NaN
  if constexpr (ACT == kGelu) {
    float e;
    return z * normal_cdf(z, e);
  }
  if constexpr (ACT == kSilu) return z / (1.f + __expf(-z));
  return z;
}

template <int ACT>
__device__ __forceinline__ float act_slope(float z) {
  if constexpr (ACT == kRelu) return z > 0.f ? 1.f : 0.f;
  if constexpr (ACT == kGelu) {
    float e;
    const float cdf = normal_cdf(z, e);
    return fmaf(z * 0.3989422804f, e, cdf);
  }
  if constexpr (ACT == kSilu) {
    const float g = 1.f / (1.f + __expf(-z));
    return g * (1.f + z * (1.f - g));
  }
  return 1.f;
}

// What an epilogue does: an Act with bias, z and residual, or nothing.
constexpr int kPlain = -1;

// the type in which z is kept
template <typename T, int ACT>
using Kept = std::conditional_t<ACT == kRelu, T, float>;

// The values of out[i][j ... j + 8), of which n exist: bias and residual are
// loaded by the caller, which has many rows of them under way.
template <typename T, int EPI>
__device__ __forceinline__ void finish(const Product& a, int64_t i, int64_t j, int n,
                                       float (&v)[8], const float (&bias)[8],
                                       s16x8 residual) {
  const int64_t at = i * a.j + j;
  if constexpr (EPI != kPlain) {
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += bias[e];
    using Z = Kept<T, EPI>;
    if (a.z) store_some<Z, 8>((Z*)a.z + at, n, v);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] = act<EPI>(v[e]);
    if (a.residual) {
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const short bits = residual[e];
        v[e] += (float)__builtin_bit_cast(T, bits);
      }
    }
  }
  if (a.out_f32) store_some<float, 8>((float*)a.out + at, n, v);
  else store_some<T, 8>((T*)a.out + at, n, v);
}

template <typename T>
__device__ __forceinline__ void load_bias(const Product& a, int64_t j, int n,
                                          float (&b)[8]) {
#pragma unroll
  for (int e = 0; e < 8; ++e) b[e] = 0.f;
  if (!a.bias || n <= 0) return;
  if (a.bias_f32) load_some<float, 8>((const float*)a.bias + j, n, b, 0.f);
  else load_some<T, 8>((const T*)a.bias + j, n, b, 0.f);
}

template <typename T>
__device__ __forceinline__ s16x8 load_residual(const Product& a, int64_t i, int64_t j,
                                               int n) {
  s16x8 r = (s16x8)0;
  if (i >= a.i || n <= 0) return r;
  const short* p = (const short*)a.residual + i * a.residual_stride + j;
  if (n >= 8) {
    __builtin_memcpy(&r, p, 16);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e)
      if (e < n) r[e] = p[e];
  }
  return r;
}

// ---- tiles

// An operand's tile of B i by KR r in LDS: rows of chunks of 8 elements. With r
// contiguous a row is one i and holds KR r; otherwise a row is one r and holds
// the tile's B values of i.
template <int B, bool TR, int KR>
struct Tile {
  static constexpr int rows = TR ? KR : B;
  static constexpr int chunks = TR ? B / 8 : KR / 8;
  static constexpr int bytes = rows * chunks * 16;

  // The chunk's place in its row. A read with r contiguous takes 16 lanes' rows
  // together, in fours of which two ask for one chunk and two for its neighbour;
  // a turning read takes 32 bytes, so there pairs of chunks move together.
  static __device__ __forceinline__ int place(int row, int chunk) {
    if constexpr (TR && B == 64)        // two rows fill the banks
      return chunk ^ ((((row >> 1) & 1) | ((row >> 2) & 2)) << 1);
    else if constexpr (TR) return chunk ^ (((row & 3) | ((row >> 1) & 4)) << 1);
    else if constexpr (KR == 32) return chunk ^ (-(row >> 2) & 3);
    else return chunk ^ ((row >> 1) & 7);
  }

  // 8 consecutive r from r0 + 8 (lane / 16) on of i = i0 + lane % 16
  static __device__ __forceinline__ s16x8 fragment(const char* lds, int i0, int r0) {
    const int lane = threadIdx.x & 63;
    if constexpr (TR) {
      // lanes 4q ... 4q + 3 of 16 fetch row q's 16 elements; lane c gets
      // column c of the 4 rows
      s16x4 part[2];
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int row = r0 + (lane >> 4) * 8 + h * 4 + ((lane >> 2) & 3);
        const int col = i0 + (lane & 3) * 4;
        const char* p = lds + (row * chunks + place(row, col >> 3)) * 16 +
                        (col & 7) * 2;
        part[h] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4)p);
      }
      return __builtin_shufflevector(part[0], part[1], 0, 1, 2, 3, 4, 5, 6, 7);
    } else {
      const int row = i0 + (lane & 15);
      const int chunk = (r0 >> 3) + (lane >> 4);
      return *(const s16x8*)(lds + (row * chunks + place(row, chunk)) * 16);
    }
  }
};

// A wave's fragments of 32 r of a tile of KR.
template <int BI, int BJ, int FI, int FJ, bool PT, bool QT, int KR>
struct Fragments {
  s16x8 p[FI], q[FJ];
  __device__ __forceinline__ void read(const char* lds, int wi, int wj, int r0 = 0) {
    using P = Tile<BI, PT, KR>;
#pragma unroll
    for (int x = 0; x < FI; ++x) p[x] = P::fragment(lds, wi + x * 16, r0);
#pragma unroll
    for (int y = 0; y < FJ; ++y)
      q[y] = Tile<BJ, QT, KR>::fragment(lds + P::bytes, wj + y * 16, r0);
  }
};

// Asks the scheduler to put one of READS LDS reads in front of each of the first
// matrix instructions. (With the reads spread evenly over all of them, or left to
// the compiler, the three bare products of 16384 x 4096 x 2048 run at 966 to 1200
// TFLOP/s, so at 1142 to 1213, one after the other of the same kind.)
template <int READS>
__device__ __forceinline__ void spread() {
#pragma unroll
  for (int i = 0; i < READS; ++i) {
    __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);                   // a read
    __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);                   // a product
  }
}

// A tile's loads by way of registers, at any alignment: each thread N chunks. A
// chunk that would pass the end of its row is loaded from further left and moved
// into place on its way to LDS, zeros behind it; so every load is made, without a
// condition, and waits can count them.
template <typename T, int B, bool TR, int NT>
struct Staged {
  using L = Tile<B, TR, kSR>;
  static constexpr int n = L::rows * L::chunks / NT;
  const T* tile;              // the same for all lanes; moves on with each tile
  int32_t offset[n];          // bytes from there; stays
  int back[n];                // elements that the load starts before its chunk (TR)
  int64_t columns;            // of a row from the tile's first on (not TR)

  static __device__ __forceinline__ int row_of(int k) {
    return (k * NT + threadIdx.x) / L::chunks;
  }
  static __device__ __forceinline__ int chunk_of(int k) {
    return (k * NT + threadIdx.x) % L::chunks;
  }

  // cols: a row's elements in memory, 8 at least
  __device__ __forceinline__ void start(const T* base, int64_t stride, int64_t i0,
                                        int64_t i_end, int64_t r0, int64_t cols) {
    tile = TR ? base + r0 * stride + i0 : base + i0 * stride + r0;
    columns = cols - r0;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const int64_t last = TR ? cols - i0 - 8 : i_end - 1 - i0;
      const int row = row_of(k), chunk = chunk_of(k);
      if constexpr (TR) {
        const int at = chunk * 8 < last ? chunk * 8 : (int)last;
        back[k] = chunk * 8 - at;
        offset[k] = (int32_t)((row * stride + at) * (int)sizeof(T));
      } else {
        const int line = row < last ? row : (int)last;
        offset[k] = (int32_t)((line * stride + chunk * 8) * (int)sizeof(T));
      }
    }
  }

  // left: how many r there are from the tile's first on; at least 1
  __device__ __forceinline__ void load(s16x8 (&v)[n], int64_t stride, int64_t left) {
    int32_t o[n];
#pragma unroll
    for (int k = 0; k < n; ++k) o[k] = offset[k];
    if (TR ? left < kSR : columns < kSR) {
#pragma unroll
      for (int k = 0; k < n; ++k) {
        if constexpr (TR) {
          const int over = row_of(k) - ((int)left - 1);
          if (over > 0) o[k] -= (int32_t)(over * stride * (int)sizeof(T));
        } else {
          const int over = chunk_of(k) * 8 - ((int)columns - 8);
          if (over > 0) o[k] -= over * (int)sizeof(T);
        }
      }
    }
#pragma unroll
    for (int k = 0; k < n; ++k) __builtin_memcpy(&v[k], (const char*)tile + o[k], 16);
  }
  __device__ __forceinline__ void next(int64_t stride) {
    tile += TR ? kSR * stride : kSR;
    columns -= kSR;
  }

  // columns_, left: of the tile that v holds
  __device__ __forceinline__ void store(const s16x8 (&v)[n], char* lds, int64_t left,
                                        int64_t columns_, bool edge) const {
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const int row = row_of(k), chunk = chunk_of(k);
      s16x8 x = v[k];
      if (TR ? edge || left < kSR : columns_ < kSR) {
        int by = TR ? back[k] : chunk * 8 - ((int)columns_ - 8);
        by = by < 0 ? 0 : by > 8 || (TR && row >= left) ? 8 : by;
        x = moved(x, by);
      }
      *(s16x8*)(lds + (row * L::chunks + L::place(row, chunk)) * 16) = x;
    }
  }

  // x[e + by], zeros behind
  static __device__ __forceinline__ s16x8 moved(s16x8 x, int by) {
    typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
    u64x2 u = __builtin_bit_cast(u64x2, x);
    uint64_t lo = u[0], hi = u[1];
    if (by & 4) lo = hi, hi = 0;
    const int bits = (by & 3) * 16;
    const uint64_t carry = bits ? hi << (64 - bits) : 0;
    u[0] = by >= 8 ? 0 : lo >> bits | carry;
    u[1] = by >= 8 ? 0 : hi >> bits;
    return __builtin_bit_cast(s16x8, u);
  }
};

// Which part of the output a block takes. Blocks go to the 8 dies in turn; each
// die gets a contiguous range of tiles, and neighbours in it form bands of 8
// tiles of i, so that blocks which run together on a die share operands in its
// cache.
struct Place {
  int i, j, split;
};
struct Tiles {
  int i, j, splits;

  __device__ __forceinline__ Place place(int block) const {
    const int total = i * j * splits;
    const int die = block & 7, each = total >> 3, more = total & 7;
    int n = block >> 3;
    n += die < more ? die * (each + 1) : more * (each + 1) + (die - more) * each;
    Place p;
    p.split = n / (i * j);
    n -= p.split * (i * j);
    const int band = n / (8 * j), rest = n - band * 8 * j;
    const int high = i - band * 8 < 8 ? i - band * 8 : 8;
    p.j = rest / high;
    p.i = band * 8 + rest - p.j * high;
    return p;
  }
};

// LDS that a wave needs to put its part of the output, XP x 16 rows at a time.
template <int FJ, int XP>
constexpr int put_bytes() { return XP * 16 * (FJ * 16 + 4) * 4; }

// A wave's part of the output from (i0, j0) on. A lane holds 4 consecutive j of
// one i of each 16 x 16; by way of LDS it gets runs of 8, so that a row's
// accesses are whole lines and the epilogue is there once.
template <typename T, int FI, int FJ, int XP, int EPI>
__device__ __forceinline__ void put(const Product& a, const f32x4 (&acc)[FI][FJ],
                                    char* lds, int split, int64_t i0, int64_t j0) {
  constexpr int kPitch = FJ * 16 + 4;        // floats; 16 rows meet no bank twice
  constexpr int kLanes = FJ * 2;             // a row's
  constexpr int kRows = 64 / kLanes;         // that a wave takes at once
  constexpr int kGroup = XP * 16 / kRows < 8 ? XP * 16 / kRows : 8;
  const int lane = threadIdx.x & 63;
  float* const part = (float*)lds;
  const int64_t j = j0 + lane % kLanes * 8;
  const int64_t left = a.j - j;
  const int n = left < 8 ? (int)left : 8;
  float bias[8];
  s16x8 residual[kGroup];                    // the group's that comes next
  const bool more = EPI != kPlain && a.residual;
  if constexpr (EPI != kPlain) load_bias<T>(a, j, n, bias);
#pragma unroll
  for (int g = 0; g < kGroup; ++g) {
    residual[g] = (s16x8)0;
    if (more) residual[g] = load_residual<T>(a, i0 + g * kRows + lane / kLanes, j, n);
  }
#pragma unroll
  for (int x = 0; x < FI; x += XP) {
#pragma unroll
    for (int u = 0; u < XP; ++u)
#pragma unroll
      for (int y = 0; y < FJ; ++y)
        *(f32x4*)(part + (u * 16 + (lane & 15)) * kPitch + y * 16 + (lane >> 4) * 4) =
            acc[x + u][y];
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
#pragma unroll 1
    for (int row0 = 0; row0 < XP * 16; row0 += kGroup * kRows) {
      s16x8 r[kGroup];
#pragma unroll
      for (int g = 0; g < kGroup; ++g) r[g] = residual[g];
      if (more) {
#pragma unroll
        for (int g = 0; g < kGroup; ++g)
          residual[g] = load_residual<T>(
              a, i0 + x * 16 + row0 + (kGroup + g) * kRows + lane / kLanes, j, n);
      }
#pragma unroll
      for (int g = 0; g < kGroup; ++g) {
        const int row = row0 + g * kRows + lane / kLanes;
        const int64_t i = i0 + x * 16 + row;
        float v[8];
        __builtin_memcpy(v, __builtin_assume_aligned(part + row * kPitch +
                                                     lane % kLanes * 8, 16), 32);
        if (i >= a.i || n <= 0) continue;
        if (EPI == kPlain && a.partial)
          store_run<float, 8>(a.partial + (split * a.i + i) * a.partial_cols + j, v);
        else
          finish<T, EPI>(a, i, j, n, v, bias, r[g]);
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
  }
}

// BI x BJ of the output by WI x WJ waves, operands at any alignment. While a tile
// is multiplied, the next one goes from registers to LDS, and the two after that are
// under way into two sets of registers. (Tiles of 32 r, four under way, take 43 us
// for 32768 x 997 by 256 where these take 39.7: a row's 128-byte line is then asked
// for twice, and the second request waits for the first.)
template <typename T, int BI, int BJ, int WI, int WJ, bool PT, bool QT, int EPI>
__global__ __launch_bounds__(WI * WJ * 64, BI * BJ < 128 * 128 ? 4 : 2)
void product_kernel(Product a, Tiles map) {
  constexpr int NT = WI * WJ * 64;
  constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16;
  constexpr int kPBytes = Tile<BI, PT, kSR>::bytes;
  constexpr int kBytes = kPBytes + Tile<BJ, QT, kSR>::bytes;
  using P = Staged<T, BI, PT, NT>;
  using Q = Staged<T, BJ, QT, NT>;
  __shared__ __attribute__((aligned(16))) char lds[2 * kBytes];
  const int wave = threadIdx.x >> 6;
  const Place at = map.place(blockIdx.x);
  const int64_t i0 = (int64_t)at.i * BI, j0 = (int64_t)at.j * BJ;
  const int wi = wave / WJ * (BI / WI), wj = wave % WJ * (BJ / WJ);
  // this block's part of r, whole tiles
  const int tiles = (int)((a.r + kSR - 1) / kSR);
  const int first = (int)((int64_t)tiles * at.split / a.splits);
  const int count = (int)((int64_t)tiles * (at.split + 1) / a.splits) - first;
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) acc[x][y] = (f32x4)0.f;
  P p;
  Q q;
  p.start((const T*)a.p, a.p_stride, i0, a.i, (int64_t)first * kSR, a.p_cols);
  q.start((const T*)a.q, a.q_stride, j0, a.j, (int64_t)first * kSR, a.q_cols);
  const bool edge_p = a.p_cols - i0 < BI, edge_q = a.q_cols - j0 < BJ;
  s16x8 vp[2][P::n], vq[2][Q::n];
  // a tile's r from its first on, and its rows' columns, as they are stored
  const int64_t left0 = a.r - (int64_t)first * kSR;
  const int64_t p_columns = p.columns, q_columns = q.columns;
  int loaded = 0;
  auto load = [&](int set) {          // the next tile, the last one for ever
    const int64_t left = left0 - (int64_t)loaded * kSR;
    p.load(vp[set], a.p_stride, left);
    q.load(vq[set], a.q_stride, left);
    if (loaded + 1 < count) {
      ++loaded;
      p.next(a.p_stride);
      q.next(a.q_stride);
    }
  };
  auto store = [&](int set, int t) {
    const int64_t done = (int64_t)t * kSR;
    p.store(vp[set], lds + set * kBytes, left0 - done, p_columns - done, edge_p);
    q.store(vq[set], lds + set * kBytes + kPBytes, left0 - done, q_columns - done, edge_q);
  };
  using F = Fragments<BI, BJ, FI, FJ, PT, QT, kSR>;
  F one, two;
  auto multiply = [&](const F& f) {
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y) acc[x][y] = mma(f.q[y], f.p[x], acc[x][y], T());
  };
  load(0);
  load(1);
  store(0, 0);
  load(0);
  // tile t lies in LDS t % 2, tile t + 1 in registers (t + 1) % 2
  auto step = [&](int t, int k) {
    __syncthreads();
    one.read(lds + k * kBytes, wi, wj, 0);
    two.read(lds + k * kBytes, wi, wj, 32);
    multiply(one);
    store(k ^ 1, t + 1);
    load(k ^ 1);
    multiply(two);
  };
  int t = 0;
  for (; t + 2 <= count; t += 2) {
    step(t, 0);
    step(t + 1, 1);
  }
  if (t < count) step(t, 0);
  __syncthreads();
  static_assert(WI * WJ * put_bytes<FJ, 2>() <= sizeof(lds), "LDS");
  put<T, FI, FJ, 2, EPI>(a, acc, lds + wave * put_bytes<FJ, 2>(), at.split, i0 + wi,
                         j0 + wj);
}

// ---- whole chunks: straight from memory into LDS

__device__ __attribute__((aligned(16))) const uint32_t kZeros[4] = {0, 0, 0, 0};

// 16 bytes for each lane from base + offset into LDS, lane after lane from `lds`
// on (the same for all lanes, as is base). Written out because behind the builtin
// the compiler waits for every load under way before it reads LDS at all; these
// loads write no register, and the kernel counts and waits for them itself.
__device__ __forceinline__ void to_lds(const void* base, uint32_t offset, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, %1"
               :: "v"(offset), "s"(base), "s"(lds) : "memory", "m0");
}
__device__ __forceinline__ void to_lds(const void* from, uint32_t lds) {
  asm volatile("s_mov_b32 m0, %1\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %0, off"
               :: "v"(from), "s"(lds) : "memory", "m0");
}

// A tile's loads where every chunk of 8 is wholly inside or outside the operand
// and aligned. A load writes 16 bytes for each of a wave's lanes, one after the
// other, so the lane whose bytes land at a place asks for the chunk that belongs
// there. Chunks behind r's end come from a block of zeros.
template <typename T, int B, bool TR, int NT>
struct Direct {
  using L = Tile<B, TR, kR>;
  static constexpr int n = L::rows * L::chunks / NT;
  const T* tile;              // the same for all lanes; moves on with each tile
  uint32_t offset[n];         // bytes from there; stays
  int64_t ahead;              // r, or a row's elements, from the tile's first on

  // cols: a row's elements in memory, a multiple of 8
  __device__ __forceinline__ void start(const T* base, int64_t stride, int64_t i0,
                                        int64_t i_end, int64_t r0, int64_t r_end,
                                        int64_t cols) {
    tile = TR ? base + r0 * stride + i0 : base + i0 * stride + r0;
    ahead = (TR ? r_end : cols < r_end + 8 ? cols : r_end) - r0;
#pragma unroll
    for (int k = 0; k < n; ++k) {
      const int slot = k * NT + threadIdx.x;
      const int row = slot / L::chunks, chunk = L::place(row, slot % L::chunks);
      int64_t at;
      if constexpr (TR) {
        const int64_t last = cols - 8 - i0;
        at = row * stride + (chunk * 8 < last ? chunk * 8 : last);
      } else {
        const int64_t last = i_end - 1 - i0;
        at = (row < last ? row : last) * stride + chunk * 8;
      }
      offset[k] = (uint32_t)(at * sizeof(T));
    }
  }

  __device__ __forceinline__ void load(uint32_t lds, int64_t stride) {
    lds += __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) * 1024;
    if (ahead >= kR) {
#pragma unroll
      for (int k = 0; k < n; ++k) to_lds(tile, offset[k], lds + k * NT * 16);
    } else {
#pragma unroll
      for (int k = 0; k < n; ++k) {
        const int slot = k * NT + threadIdx.x;
        const int row = slot / L::chunks, chunk = L::place(row, slot % L::chunks);
        const char* p = (TR ? row : chunk * 8) < ahead ? (const char*)tile + offset[k]
                                                       : (const char*)kZeros;
        to_lds(p, lds + k * NT * 16);
      }
    }
    tile += TR ? kR * stride : kR;
    ahead -= kR;
  }
};

// S tiles of LDS under way and two sets of fragments, one multiplied while the
// other is read. A step's barrier says that the next tile has arrived, and that
// this one is in registers, so that its LDS can take the tile S further on. Every
// step loads a tile, zeros behind r's end, so that a fixed number of loads is under
// way and a wait can leave the youngest S - 2 tiles' alone. 256 x 256 takes four
// tiles and a compute unit, 128 x 128 three and 64 x 64 six, so that three blocks
// share one.
template <typename T, int BI, int BJ, int WI, int WJ, bool PT, bool QT, int EPI>
__global__ __launch_bounds__(WI * WJ * 64, BI * BJ > 128 * 128 ? 1 : 3)
void product_direct_kernel(Product a, Tiles map) {
  constexpr int S = BI * BJ > 128 * 128 ? 4 : BI * BJ < 128 * 128 ? 6 : 3;
  constexpr int NT = WI * WJ * 64;
  constexpr int FI = BI / WI / 16, FJ = BJ / WJ / 16;
  constexpr int kReads = (PT ? 2 : 1) * FI + (QT ? 2 : 1) * FJ;
  constexpr int kPBytes = Tile<BI, PT, kR>::bytes;
  constexpr int kBytes = kPBytes + Tile<BJ, QT, kR>::bytes;
  constexpr int kLoads = Direct<T, BI, PT, NT>::n + Direct<T, BJ, QT, NT>::n;
  // s_waitcnt: at most S - 2 tiles' loads under way, no LDS read
  constexpr int kLeave = (S - 2) * kLoads, kFirst = (S - 1) * kLoads;
  constexpr int kWait = (kLeave & 15) | (kLeave >> 4) << 14 | 7 << 4;
  constexpr int kWaitFirst = (kFirst & 15) | (kFirst >> 4) << 14 | 7 << 4;
  static_assert(kFirst < 64, "waits");
  __shared__ __attribute__((aligned(16))) char lds[S * kBytes];
  const int wave = threadIdx.x >> 6;
  const Place at = map.place(blockIdx.x);
  const int64_t i0 = (int64_t)at.i * BI, j0 = (int64_t)at.j * BJ;
  const int wi = wave / WJ * (BI / WI), wj = wave % WJ * (BJ / WJ);
  const int tiles = (int)((a.r + kR - 1) / kR);
  const int first = (int)((int64_t)tiles * at.split / a.splits);
  const int count = (int)((int64_t)tiles * (at.split + 1) / a.splits) - first;
  f32x4 acc[FI][FJ];
#pragma unroll
  for (int x = 0; x < FI; ++x)
#pragma unroll
    for (int y = 0; y < FJ; ++y) acc[x][y] = (f32x4)0.f;
  Direct<T, BI, PT, NT> p;
  Direct<T, BJ, QT, NT> q;
  // another block's tiles are loaded behind the last one, and not used
  p.start((const T*)a.p, a.p_stride, i0, a.i, (int64_t)first * kR, a.r, a.p_cols);
  q.start((const T*)a.q, a.q_stride, j0, a.j, (int64_t)first * kR, a.r, a.q_cols);
  const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char*)lds;
  int stage = 0;                                         // the next load's
  auto load = [&]() {
    p.load(lds0 + stage, a.p_stride);
    q.load(lds0 + stage + kPBytes, a.q_stride);
    stage = stage == (S - 1) * kBytes ? 0 : stage + kBytes;
  };
  using F = Fragments<BI, BJ, FI, FJ, PT, QT, kR>;
  int ready = kBytes;                                    // the tile to read next
  auto step = [&](const F& now, F& next) {
    __builtin_amdgcn_s_waitcnt(kWait);
    __syncthreads();
    load();
    next.read(lds + ready, wi, wj);
    ready = ready == (S - 1) * kBytes ? 0 : ready + kBytes;
#pragma unroll
    for (int x = 0; x < FI; ++x)
#pragma unroll
      for (int y = 0; y < FJ; ++y) acc[x][y] = mma(now.q[y], now.p[x], acc[x][y], T());
    spread<kReads>();
  };
  F one, two;
#pragma unroll 1
  for (int k = 0; k < S; ++k) load();
  __builtin_amdgcn_s_waitcnt(kWaitFirst);
  __syncthreads();
  one.read(lds, wi, wj);
  int t = 0;
  for (; t + 2 <= count; t += 2) {
    step(one, two);
    step(two, one);
  }
  if (t < count) step(one, two);
  __builtin_amdgcn_s_waitcnt(0);
  __syncthreads();
  static_assert(WI * WJ * put_bytes<FJ, 2>() <= sizeof(lds), "LDS");
  put<T, FI, FJ, 2, EPI>(a, acc, lds + wave * put_bytes<FJ, 2>(), at.split, i0 + wi, j0 + wj);
}

// The parts of r added up, and the epilogue. G threads take every G-th part of 8
// values of the output, and their sums are added up in a fixed order.
template <typename T, int EPI, int G>
__global__ __launch_bounds__(256) void product_join_kernel(Product a) {
  constexpr int R = 256 / G;
  __shared__ float lds[G > 1 ? 256 : 1][8];
  const int64_t runs = (a.j + 7) / 8;
  const int64_t at = (int64_t)blockIdx.x * R + threadIdx.x % R;
  const int group = threadIdx.x / R;
  const bool some = at < a.i * runs;
  const int64_t i = some ? at / runs : 0, j = some ? at % runs * 8 : 0;
  const int n = a.j - j < 8 ? (int)(a.j - j) : 8;
  float bias[8], v[8] = {};
  s16x8 residual = (s16x8)0;
  if constexpr (EPI != kPlain) {
    load_bias<T>(a, j, n, bias);
    if (a.residual) residual = load_residual<T>(a, i, j, n);
  }
  const float* p = a.partial + i * a.partial_cols + j;
  const int64_t part = a.i * a.partial_cols;
#pragma unroll 4
  for (int s = group; s < a.splits; s += G) {
    float q[8];
    load_run<float, 8>(p + s * part, q);
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += q[e];
  }
  if constexpr (G > 1) {
    store_run<float, 8>(lds[threadIdx.x], v);
    __syncthreads();
    if (group) return;
    for (int g = 1; g < G; ++g)
#pragma unroll
      for (int e = 0; e < 8; ++e) v[e] += lds[g * R + threadIdx.x][e];
  }
  if (some) finish<T, EPI>(a, i, j, n, v, bias, residual);
}

// ---- few rows

constexpr int kFewWaves = 8;

// 16 columns of the output for at most MT x 16 rows: what bounds a layer with few
// rows is how soon its weights arrive, so each of 8 waves asks for an eighth of r
// of both operands straight into fragments, and the waves' sums meet in LDS. One
// launch, and no parts to join: 16 x 1024 by 256 takes 4.6 us, by tiles of 64
// with r in 4 parts 9.4 us.
template <typename T, int MT, int EPI>
__global__ __launch_bounds__(kFewWaves * 64)
void product_few_kernel(Product a) {
  __shared__ __attribute__((aligned(16))) float part[kFewWaves][MT * 16][16];
  constexpr int kAhead = MT > 2 ? 2 : 4;      // steps of 32 r under way together
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
  const int64_t j0 = (int64_t)blockIdx.x * 16;
  const int64_t j = j0 + (lane & 15) < a.j ? j0 + (lane & 15) : a.j - 1;
  const T* q = (const T*)a.q + j * a.q_stride;
  const T* p[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) {
    const int64_t i = m * 16 + (lane & 15);
    p[m] = (const T*)a.p + (i < a.i ? i : a.i - 1) * a.p_stride;
  }
  f32x4 acc[MT];
#pragma unroll
  for (int m = 0; m < MT; ++m) acc[m] = (f32x4)0.f;
  const int chunk = (lane >> 4) * 8;
  // 8 elements from r on; the last ones of a row by way of those before them
  auto load = [&](const T* row, int64_t r, int64_t cols) {
    s16x8 v;
    const int64_t at = r < cols - 8 ? r : cols - 8;
    __builtin_memcpy(&v, row + at, 16);
    return v;
  };
  auto placed = [&](s16x8 v, int64_t r, int64_t cols) {
    const int64_t by = r - (cols - 8);
    return by > 0 ? Staged<T, 128, false, 256>::moved(v, by < 8 ? (int)by : 8) : v;
  };
  for (int64_t r0 = wave * 32; r0 < a.r; r0 += kFewWaves * 32 * kAhead) {
    s16x8 fq[kAhead], fp[kAhead][MT];
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t r = r0 + k * kFewWaves * 32 + chunk;
      fq[k] = load(q, r, a.q_cols);
#pragma unroll
      for (int m = 0; m < MT; ++m) fp[k][m] = load(p[m], r, a.p_cols);
    }
#pragma unroll
    for (int k = 0; k < kAhead; ++k) {
      const int64_t r = r0 + k * kFewWaves * 32 + chunk;
      fq[k] = placed(fq[k], r, a.q_cols);
#pragma unroll
      for (int m = 0; m < MT; ++m)
        acc[m] = mma(fq[k], placed(fp[k][m], r, a.p_cols), acc[m], T());
    }
  }
#pragma unroll
  for (int m = 0; m < MT; ++m)
    *(f32x4*)&part[wave][m * 16 + (lane & 15)][(lane >> 4) * 4] = acc[m];
  __syncthreads();
  const int64_t i = threadIdx.x >> 1, at = j0 + (threadIdx.x & 1) * 8;
  if (i >= a.i || at >= a.j || i >= MT * 16) return;
  const int n = a.j - at < 8 ? (int)(a.j - at) : 8;
  float bias[8], v[8] = {};
  s16x8 residual = (s16x8)0;
  if constexpr (EPI != kPlain) {
    load_bias<T>(a, at, n, bias);
    if (a.residual) residual = load_residual<T>(a, i, at, n);
  }
#pragma unroll
  for (int w = 0; w < kFewWaves; ++w)
#pragma unroll
    for (int e = 0; e < 8; ++e) v[e] += part[w][i][(threadIdx.x & 1) * 8 + e];
  finish<T, EPI>(a, i, at, n, v, bias, residual);
}

// ---- dz and db

constexpr int kActRows = 4;           // rows of a thread under way together

template <typename T>
__device__ __forceinline__ void put_dbias(const ActBwd& a, int64_t c, float v) {
  if (a.dbias_f32) ((float*)a.dbias)[c] = v;
  else ((T*)a.dbias)[c] = (T)v;
}

// 32 threads take 8 columns each, 8 rows at a time. NARROW: fewer than 8 columns.
template <typename T, int ACT, bool NARROW>
__global__ __launch_bounds__(256) void act_bwd_kernel(ActBwd a) {
  __shared__ float part[8][257];
  const int t = threadIdx.x & 31, group = threadIdx.x >> 5;
  const RowRun<T, NARROW> run(blockIdx.x * 256 + t * 8, (int)a.n);
  float db[8] = {};
  if (run.any())
    for (int64_t i0 = (int64_t)blockIdx.y * 8 * kActRows + group; i0 < a.rows;
         i0 += (int64_t)gridDim.y * 8 * kActRows) {
      float d[kActRows][8], z[kActRows][8];
#pragma unroll
      for (int k = 0; k < kActRows; ++k) {
        const int64_t i = i0 + k * 8 < a.rows ? i0 + k * 8 : a.rows - 1;
        run.load((const T*)a.dy + i * a.dy_stride, d[k]);
        if constexpr (ACT != kNone) run.load((const Kept<T, ACT>*)a.z + i * a.n, z[k]);
      }
#pragma unroll
      for (int k = 0; k < kActRows; ++k) {
        if (i0 + k * 8 >= a.rows) break;
        if constexpr (ACT != kNone) {
#pragma unroll
          for (int e = 0; e < 8; ++e) {
            if constexpr (ACT == kRelu)
              d[k][e] = z[k][e] > 0.f ? d[k][e] : z[k][e] != z[k][e] ? z[k][e] : 0.f;
            else
              d[k][e] *= act_slope<ACT>(z[k][e]);
          }
          run.store((T*)a.dz + (i0 + k * 8) * a.n, d[k]);
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) db[e] += d[k][e];
      }
    }
  if (!a.dbias) return;
  // the run that moved back has some columns twice
#pragma unroll
  for (int e = 0; e < 8; ++e)
    if (run.counts(e)) part[group][run.at + e - blockIdx.x * 256] = db[e];
  __syncthreads();
  const int64_t col = (int64_t)blockIdx.x * 256 + threadIdx.x;
  if (col >= a.n) return;
  float v = 0.f;
#pragma unroll
  for (int g = 0; g < 8; ++g) v += part[g][threadIdx.x];
  if (a.partial) a.partial[blockIdx.y * a.n + col] = v;
  else put_dbias<T>(a, col, v);
}

template <typename T>
__global__ __launch_bounds__(1024) void bias_join_kernel(ActBwd a) {
  __shared__ float lds[64][17];
  const int lane = threadIdx.x % 16, group = threadIdx.x / 16;
  const int64_t c = (int64_t)blockIdx.x * 16 + lane;
  float v = 0.f;
  if (c < a.n)
#pragma unroll 4
    for (int k = group; k < a.blocks; k += 64) v += a.partial[k * a.n + c];
  lds[group][lane] = v;
  __syncthreads();
  if (group == 0 && c < a.n) {
    for (int k = 1; k < 64; ++k) v += lds[k][lane];
    put_dbias<T>(a, c, v);
  }
}

int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

// Whether an operand's rows are whole aligned chunks of 8, and a tile's offsets
// fit 32 bits.
bool chunked(const void* p, int64_t stride, int64_t cols) {
  return ((uintptr_t)p & 15) == 0 && stride % 8 == 0 && stride < (1 << 22) &&
         cols % 8 == 0;
}

bool direct(const Product& a) {
  return chunked(a.p, a.p_stride, a.p_cols) && chunked(a.q, a.q_stride, a.q_cols);
}

// A wave's next loads wait for its last ones, so long rows go by tiles, with r in
// parts: 64 x 1024 by 256 takes 7.2 us here, 9.6 by tiles; 64 x 4096 by 4096 21 and
// 16; 16 x 4096 by 4096 11 and 15; 16 x 8192 by 1024 17 and 11. Unaligned rows cost
// more here: 16 x 997 by 301 6.8 and 9.5, 16 x 2001 by 301 12.4 and 10.6.
bool few(const Product& a) {
  if (a.p_t || a.q_t || a.i > 64) return false;
  return a.r <= (!direct(a) ? 1024 : a.i <= 32 ? 4096 : 2048);
}

// Tiles of 256 x 256, of which one fills a compute unit, need 1024 r to outweigh
// their first loads (bare, 16384 x 1024 by 4096 takes 156 us by tiles of 128, 149 us
// by these; 32768 x 1000 by 256 31 and 48) and 2048 where nothing hides an activation
// behind them (with gelu 181 and 205; 8192 x 2048 by 2048 86 and 82, with a residual
// and z kept 104 and 91), and either enough of them for all compute units or enough r
// to share a tile among two blocks.
bool large(const Product& a) {
  const int64_t tiles = ceil_div(a.i, 256) * ceil_div(a.j, 256);
  return direct(a) && ((a.r >= (a.act ? 2048 : 1024) && tiles >= 192) || (a.r >= 4096 && tiles >= 96));
}

struct Plan {
  int side, splits;
};

// The side of the tiles and the parts of r. Of tiles of 64 and of 128 with r in 1
// to 512 parts it takes those that should end first, by what a block's steps of 32
// r take where it is alone on its compute unit (at least `alone`) and for each
// block that shares it (`shared`), and by the joining of parts: a launch, 8 bytes
// of traffic for each value of a part, and a wait for each batch of parts. The
// figures, in us, are fitted to timed products. Of 162 products of 1 to 131072 rows
// (profiles/block_ops_linear_tiles.csv: each with either side and every number of
// parts) the choice is on average 0.7% slower than the best, at worst 21%. (In us, as
// chosen and by tiles of 128 with parts for two blocks a compute unit: 512 x 1024 by
// 1024 10.7 and 26.4, 2048 x 997 by 256 10.0 and 24.7, 16384 x 256 by 256 9.1 and 27.1.)
Plan plan(const Product& a) {
  if (large(a)) {
    const int64_t tiles = ceil_div(a.i, 256) * ceil_div(a.j, 256);
    return {256, tiles <= 128 ? 2 : 1};
  }
  struct Cost {
    int side;
    double once, alone, shared;
  };
  static constexpr Cost costs[2][2] = {{{64, 2.5, 0.23, 0.22}, {128, 3.5, 0.55, 0.32}},
                                       {{64, 2.7, 0.16, 0.14}, {128, 2.9, 0.26, 0.23}}};
  const bool whole = direct(a);
  Plan best = {128, 1};
  double least = 1e30;
  for (const Cost& c : costs[whole]) {
    const int64_t tiles = ceil_div(a.i, c.side) * ceil_div(a.j, c.side);
    const int64_t deep = ceil_div(a.r, whole ? kR : kSR);
    for (int s : {1, 2, 3, 4, 6, 8, 12, 16, 24, 32, 64, 128, 256, 512}) {
      if (s > 1 && (s * 64 > a.r || tiles * s > 1024)) break;
      const double steps = (double)ceil_div(deep, s) * (whole ? 1 : 2);
      const double share = c.shared * (double)(tiles * s) / 256;
      double t = c.once + steps * (share > c.alone ? share : c.alone);
      if (s > 1)
        t += 2.3 + 8e-6 / 5.5 * (double)a.i * (double)a.j * s +
             0.64 * (double)ceil_div(s, s >= 64 ? 128 : s >= 8 ? 32 : 4);
      if (t < least) {
        least = t;
        best = {c.side, s};
      }
    }
  }
  return best;
}

template <typename T, bool PT, bool QT, int EPI>
void launch(const Product& a, hipStream_t stream) {
  if constexpr (!PT && !QT) {
    if (few(a)) {
      const dim3 grid((unsigned)ceil_div(a.j, 16));
      if (a.i <= 16) product_few_kernel<T, 1, EPI><<<grid, kFewWaves * 64, 0, stream>>>(a);
      else if (a.i <= 32) product_few_kernel<T, 2, EPI><<<grid, kFewWaves * 64, 0, stream>>>(a);
      else product_few_kernel<T, 4, EPI><<<grid, kFewWaves * 64, 0, stream>>>(a);
      return;
    }
  }
  const int side = plan(a).side;
  const Tiles map = {(int)ceil_div(a.i, side), (int)ceil_div(a.j, side), a.splits};
  const dim3 grid((unsigned)map.i * map.j * map.splits);
  if (side == 256)
    product_direct_kernel<T, 256, 256, 2, 2, PT, QT, EPI><<<grid, 256, 0, stream>>>(a, map);
  else if (direct(a) && side == 128)
    product_direct_kernel<T, 128, 128, 2, 2, PT, QT, EPI><<<grid, 256, 0, stream>>>(a, map);
  else if (direct(a))
    product_direct_kernel<T, 64, 64, 2, 2, PT, QT, EPI><<<grid, 256, 0, stream>>>(a, map);
  else if (side == 128)
    product_kernel<T, 128, 128, 2, 2, PT, QT, EPI><<<grid, 256, 0, stream>>>(a, map);
  else
    product_kernel<T, 64, 64, 2, 2, PT, QT, EPI><<<grid, 256, 0, stream>>>(a, map);
}

template <typename T, int EPI>
void join(const Product& a, hipStream_t stream) {
  const int64_t runs = a.i * ceil_div(a.j, 8);
  if (a.splits >= 64)
    product_join_kernel<T, EPI, 32><<<dim3((unsigned)ceil_div(runs, 8)), 256, 0, stream>>>(a);
  else if (a.splits >= 8)
    product_join_kernel<T, EPI, 8><<<dim3((unsigned)ceil_div(runs, 32)), 256, 0, stream>>>(a);
  else
    product_join_kernel<T, EPI, 1><<<dim3((unsigned)ceil_div(runs, 256)), 256, 0, stream>>>(a);
}

template <typename T>
void launch_any(const Product& a, hipStream_t stream) {
  const bool plain = !a.bias && !a.z && !a.act && !a.residual;
  if (a.p_t) launch<T, true, true, kPlain>(a, stream);
  else if (a.q_t) launch<T, false, true, kPlain>(a, stream);
  else if (plain || a.partial) launch<T, false, false, kPlain>(a, stream);
  else if (a.act == kNone) launch<T, false, false, kNone>(a, stream);
  else if (a.act == kRelu) launch<T, false, false, kRelu>(a, stream);
  else if (a.act == kGelu) launch<T, false, false, kGelu>(a, stream);
  else launch<T, false, false, kSilu>(a, stream);
  if (!a.partial) return;
  if (plain) join<T, kPlain>(a, stream);
  else if (a.act == kNone) join<T, kNone>(a, stream);
  else if (a.act == kRelu) join<T, kRelu>(a, stream);
  else if (a.act == kGelu) join<T, kGelu>(a, stream);
  else join<T, kSilu>(a, stream);
}

template <typename T>
void launch_act_bwd(const ActBwd& a, hipStream_t stream) {
  const dim3 grid((unsigned)ceil_div(a.n, 256), a.blocks);
  auto run = [&](auto narrow) {
    constexpr bool N = decltype(narrow)::value;
    if (a.act == kNone) act_bwd_kernel<T, kNone, N><<<grid, 256, 0, stream>>>(a);
    else if (a.act == kRelu) act_bwd_kernel<T, kRelu, N><<<grid, 256, 0, stream>>>(a);
    else if (a.act == kGelu) act_bwd_kernel<T, kGelu, N><<<grid, 256, 0, stream>>>(a);
    else act_bwd_kernel<T, kSilu, N><<<grid, 256, 0, stream>>>(a);
  };
  if (a.n < 8) run(std::true_type());
  else run(std::false_type());
  if (a.partial)
    bias_join_kernel<T><<<dim3((unsigned)ceil_div(a.n, 16)), 1024, 0, stream>>>(a);
}

}  // namespace

int product_splits(const Product& a) { return few(a) ? 1 : plan(a).splits; }

void product(const Product& a, int dtype, hipStream_t stream) {
  if (dtype == kBF16) launch_any<bf16>(a, stream);
  else launch_any<f16>(a, stream);
}

// Up to 64 rows are one block's, which needs no partial sums and no second launch:
// 33 x 256 takes 4.2 us so, 5.8 us in two blocks and a join; 128 x 256 9.2 and 5.9.
int act_bwd_blocks(int64_t rows, int64_t n) {
  if (rows <= 64) return 1;
  const int64_t wide = ceil_div(n, 256);
  int64_t b = 1024 / wide;
  b = b < 64 ? 64 : b;
  const int64_t need = ceil_div(rows, 8 * kActRows);
  return (int)(need < b ? need : b);
}

void act_bwd(const ActBwd& a, int dtype, hipStream_t stream) {
  if (dtype == kBF16) launch_act_bwd<bf16>(a, stream);
  else launch_act_bwd<f16>(a, stream);
}

}  // namespace blk
