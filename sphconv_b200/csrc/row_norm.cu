// Norms before and after a block, fused with the block's gate and residual scale, and the gradients of all of it.
//
//   inner  = norm(block) * weight + bias            (inner = block without a weight)
//   out    = residual + scale[c] * sigmoid(gate) * inner
//   normed = norm(out) * next_weight + next_bias    (from the sum before it is rounded)
//   norm(x) = x / sqrt(mean(x^2) + eps), or (x - mean(x)) / sqrt(var(x) + eps) with CENTER
//
// One pass: a row is read once into registers, by 1 to 512 threads that hold E values each, reduced among them (shuffles, or shared
// memory where they are more than a warp) and written.  Statistics and sums are float32; rows are rounded once.  A thread has its columns'
// parameters in registers and asks for its next row in front of the work on this one; what is between it and HBM's rate is then the
// number of its instructions, so values go two to a float32 operation.
// The variance is the mean of squared deviations, which the values in registers make as cheap as the mean of squares.
//
// Backward reads the block, the residual, the gate and the two gradients, makes `out` again in float32 (the rounded one would shift
// the gradient of a 16-bit row's norm) and takes mean and 1/deviation of both norms from the forward pass (16 bytes a row).  The
// threads of a persistent grid own columns, so the sums over rows - gradients of weights, biases and the scale - stay in registers
// (in shared memory with 16 values a thread: 2048 float32 rows of 8192 channels 275 -> 187 us) until the end; each block leaves its
// sums in the scratch, and a second launch adds those up in a fixed order: no atomics, the same bits every time.
#include <algorithm>

#include "common.cuh"

namespace sph {

namespace {

constexpr int kBlock = 256;                   // threads of a block where a row takes a warp or less
constexpr int kMaxWarps = 16;                 // of a row
constexpr int kSums = 5;                      // sums over rows: weight, bias, scale, next_weight, next_bias

struct Params {
  const void *block, *residual, *gate;        // [n, c], [n, c], [n, c] or [n]; block and gate may be null
  const void* param[kSums];                   // weight, bias, scale, next_weight, next_bias [c]: any may be null
  int param_dtype[kSums];
  const void *d_out, *d_normed;               // backward: either may be null
  void *out, *normed;                         // forward: either may be null
  void *d_block, *d_residual, *d_gate;        // backward: any may be null
  float* stats;                               // [n][4]: mean and 1/deviation of block and of out; null: not wanted
  float* partial;                             // backward: [blocks][kSums][c]
  int64_t n;
  int c, lanes, gate_row;                     // lanes: threads of a row, a power of two
  float eps;
};

// Rows are loaded and kept as words of their bits: 16 bytes, or one element, a piece.
template <typename T> struct Row;
template <> struct Row<float> {
  static constexpr int kVec = 4;
  using Bits = uint32_t;
  static __device__ __forceinline__ float get(uint32_t v) { return __uint_as_float(v); }
  static __device__ __forceinline__ uint32_t put(float v) { return __float_as_uint(v); }
};
template <> struct Row<__half> {
  static constexpr int kVec = 8;
  using Bits = uint16_t;
  static __device__ __forceinline__ float get(uint16_t v) { return __half2float(__ushort_as_half(v)); }
  static __device__ __forceinline__ uint16_t put(float v) { return __half_as_ushort(__float2half_rn(v)); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return __half22float2(*(const __half2*)&w); }
  static __device__ __forceinline__ uint32_t pack(float2 x) {
    const __half2 h = __float22half2_rn(x);
    return *(const uint32_t*)&h;
  }
};
template <> struct Row<__nv_bfloat16> {
  static constexpr int kVec = 8;
  using Bits = uint16_t;
  static __device__ __forceinline__ float get(uint16_t v) { return __uint_as_float((uint32_t)v << 16); }
  static __device__ __forceinline__ uint16_t put(float v) { return __bfloat16_as_ushort(__float2bfloat16_rn(v)); }
  static __device__ __forceinline__ float2 unpack(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static __device__ __forceinline__ uint32_t pack(float2 x) {
    const __nv_bfloat162 h = __float22bfloat162_rn(x);
    return *(const uint32_t*)&h;
  }
};

// A thread's values of a row: NV pieces of VEC consecutive ones, piece j at (j * lanes + t) * VEC; in pairs for the arithmetic.
template <typename T, int VEC, int NV>
struct Tile {
  static constexpr int E = VEC * NV;
  using R = Row<T>;
  using Bits = typename R::Bits;
  static constexpr int kWords = VEC > 1 ? 4 : 1;
  struct Raw { uint32_t w[NV][kWords]; };     // as they lie in memory

  static __device__ __forceinline__ int column(int j, int t, int lanes) { return (j * lanes + t) * VEC; }

  static __device__ __forceinline__ void fetch(Raw& r, const void* base, int64_t row, int c, int t, int lanes, bool active) {
    const Bits* p = (const Bits*)base + row * c;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = column(j, t, lanes);
      const bool some = active && at < c;     // c is a multiple of VEC
      if constexpr (VEC > 1) {
        const uint4 q = some ? *(const uint4*)(p + at) : make_uint4(0u, 0u, 0u, 0u);
        r.w[j][0] = q.x; r.w[j][1] = q.y; r.w[j][2] = q.z; r.w[j][3] = q.w;
      } else {
        r.w[j][0] = some ? (uint32_t)p[at] : 0u;
      }
    }
  }
  static constexpr int P = E / 2;             // pairs
  using Pairs = float2[P];
  // piece and place in it of value e
  static __device__ __forceinline__ bool inside(int e, int c, int t, int lanes) { return column(e / VEC, t, lanes) < c; }

  static __device__ __forceinline__ void values(Pairs& x, const Raw& r) {
#pragma unroll
    for (int k = 0; k < P; ++k) {
      const int e = 2 * k;
      if constexpr (VEC == 1) x[k] = make_float2(R::get((Bits)r.w[e][0]), R::get((Bits)r.w[e + 1][0]));
      else if constexpr (VEC == 4) x[k] = make_float2(__uint_as_float(r.w[e / 4][e % 4]), __uint_as_float(r.w[e / 4][e % 4 + 1]));
      else x[k] = R::unpack(r.w[e / 8][e % 8 / 2]);
    }
  }
  static __device__ __forceinline__ void store(const Pairs& x, void* base, int64_t row, int c, int t, int lanes, bool active) {
    Bits* p = (Bits*)base + row * c;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = column(j, t, lanes);
      if (!active || at >= c) continue;
      if constexpr (VEC == 1)
        p[at] = R::put(j % 2 ? x[j / 2].y : x[j / 2].x);
      else if constexpr (VEC == 4)
        *(uint4*)(p + at) = make_uint4(__float_as_uint(x[2 * j].x), __float_as_uint(x[2 * j].y), __float_as_uint(x[2 * j + 1].x),
                                       __float_as_uint(x[2 * j + 1].y));
      else
        *(uint4*)(p + at) = make_uint4(R::pack(x[4 * j]), R::pack(x[4 * j + 1]), R::pack(x[4 * j + 2]), R::pack(x[4 * j + 3]));
    }
  }
  // a parameter [c] of float32 or of 16 bits, or `other` where there is none; 16-byte aligned where rows come in pieces
  static __device__ __forceinline__ void param(Pairs& x, const void* p, int dtype, float other, int c, int t, int lanes) {
    auto wide = [&](uint32_t bits) { return dtype == SPH_F16 ? __half2float(__ushort_as_half((unsigned short)bits)) : __uint_as_float(bits << 16); };
#pragma unroll
    for (int k = 0; k < P; ++k) x[k] = make_float2(other, other);
    if (p == nullptr) return;
#pragma unroll
    for (int j = 0; j < NV; ++j) {
      const int at = column(j, t, lanes);
      if (at >= c) continue;
      if constexpr (VEC > 1) {
#pragma unroll
        for (int i = 0; i < VEC; i += 4) {
          float2 &a = x[(j * VEC + i) / 2], &b = x[(j * VEC + i) / 2 + 1];
          if (dtype == SPH_F32) {
            const float4 f = __ldg((const float4*)((const float*)p + at + i));
            a = make_float2(f.x, f.y);
            b = make_float2(f.z, f.w);
          } else {
            const uint2 h = __ldg((const uint2*)((const unsigned short*)p + at + i));
            a = make_float2(wide(h.x & 0xffffu), wide(h.x >> 16));
            b = make_float2(wide(h.y & 0xffffu), wide(h.y >> 16));
          }
        }
      } else {
        const float v = dtype == SPH_F32 ? __ldg((const float*)p + at) : wide(__ldg((const unsigned short*)p + at));
        if (j % 2) x[j / 2].y = v; else x[j / 2].x = v;
      }
    }
  }
};

__device__ __forceinline__ float2 pair(float v) { return make_float2(v, v); }
__device__ __forceinline__ float both(float2 v) { return v.x + v.y; }

// Sums over the threads of a row, in every one of them.  More than a warp: the block is one row, and calls alternate between two
// places in shared memory, so that one barrier a call is enough.
struct Reducer {
  float (*slots)[kMaxWarps][4];               // [2][warps][4]
  int lanes, turn;
  template <int N>
  __device__ __forceinline__ void sum(float (&v)[N]) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      if (2 * o > lanes) continue;            // the same for all threads
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
    }
    if (lanes > 32) {
      const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, warps = lanes >> 5;
      if (lane == 0) {
#pragma unroll
        for (int i = 0; i < N; ++i) slots[turn][warp][i] = v[i];
      }
      __syncthreads();
#pragma unroll
      for (int i = 0; i < N; ++i) v[i] = slots[turn][lane & (warps - 1)][i];
#pragma unroll
      for (int o = kMaxWarps / 2; o > 0; o >>= 1) {
        if (2 * o > warps) continue;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] += __shfl_xor_sync(0xffffffffu, v[i], o);
      }
      turn ^= 1;
    }
  }
};

// mean and 1/deviation of a row, whose values behind the end are zeros
template <typename X, bool CENTER>
__device__ __forceinline__ void statistics(const typename X::Pairs& x, Reducer& red, int c, int t, float eps, float& mean, float& inv) {
  const float per_c = 1.f / (float)c;
  mean = 0.f;
  float s[1];
  float2 a = pair(0.f);
  if (CENTER) {
#pragma unroll
    for (int k = 0; k < X::P; ++k) a = add2(a, x[k]);
    s[0] = both(a);
    red.sum(s);
    mean = s[0] * per_c;
    a = pair(0.f);
  }
#pragma unroll
  for (int k = 0; k < X::P; ++k) {
    float2 d = x[k];
    if (CENTER) {
      d = add2(d, pair(-mean));
      if (!X::inside(2 * k, c, t, red.lanes)) d.x = 0.f;
      if (!X::inside(2 * k + 1, c, t, red.lanes)) d.y = 0.f;
    }
    a = fma2(d, d, a);
  }
  s[0] = both(a);
  red.sum(s);
  inv = rsqrtf(fmaf(s[0], per_c, eps));
}

// The mean goes off first: x inv - mean inv in one operation would leave mean inv 2^-24 of a deviation that is zero (rows of 1000.1: up to 0.03).
template <bool CENTER>
__device__ __forceinline__ float2 normalised(float2 x, float mean, float inv) { return mul2(CENTER ? add2(x, pair(-mean)) : x, pair(inv)); }

// The reciprocal (of 1 and more) is off by 2^-23; 16-bit rows round what is left to 8 or 11 bits, and take a fast exponential too, that is
// off by |x| 2^-23 about.  Neither minds an exponential that is infinite.
template <typename T>
__device__ __forceinline__ float sigmoid(float x) {
  float e, y;
  if (sizeof(T) == 2) asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"(x * -1.4426950408889634f));
  else e = expf(-x);
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(1.f + e));
  return y;
}
template <typename T>
__device__ __forceinline__ float2 sigmoid(float2 x) { return make_float2(sigmoid<T>(x.x), sigmoid<T>(x.y)); }

// Blocks of an SM: what their registers have room for, backward with the sums over rows in them.  Each keeps a row on its way (rows of 64
// bf16 channels, three blocks forward instead of two: 85 -> 75 us).
constexpr int forward_blocks_per_sm(int threads) { return threads >= 512 ? 1 : 768 / threads; }
constexpr int backward_blocks_per_sm(int threads) { return threads >= 512 ? 1 : 512 / threads; }

// BIAS: there may be biases.  THREADS: most threads of a block.
template <typename T, int VEC, int NV, bool CENTER, bool BIAS, int THREADS>
__global__ void __launch_bounds__(THREADS, forward_blocks_per_sm(THREADS)) forward_kernel(const __grid_constant__ Params p) {
  using X = Tile<T, VEC, NV>;
  constexpr int P = X::P;
  using Pairs = typename X::Pairs;
  __shared__ float slots[2][kMaxWarps][4];
  after_previous();
  const int lanes = p.lanes, c = p.c, t = threadIdx.x & (lanes - 1), rows = blockDim.x / lanes;
  const bool gated = p.gate && !p.gate_row;
  Reducer red{slots, lanes, 0};
  Pairs weight, scale, next_weight;
  X::param(weight, p.param[0], p.param_dtype[0], 1.f, c, t, lanes);
  X::param(scale, p.param[2], p.param_dtype[2], 1.f, c, t, lanes);
  X::param(next_weight, p.param[3], p.param_dtype[3], 1.f, c, t, lanes);
  typename X::Raw raw_x, raw_b, raw_g;
  typename Row<T>::Bits raw_rg = 0;
  auto fetch = [&](int64_t row) {
    const bool some = row < p.n;
    X::fetch(raw_x, p.residual, row, c, t, lanes, some);
    if (p.block) X::fetch(raw_b, p.block, row, c, t, lanes, some);
    if (gated) X::fetch(raw_g, p.gate, row, c, t, lanes, some);
    else if (p.gate && some) raw_rg = ((const typename Row<T>::Bits*)p.gate)[row];
  };
  const int64_t first = (int64_t)blockIdx.x * rows, step = (int64_t)gridDim.x * rows;
  const int mine = threadIdx.x / lanes;
  if (first < p.n) fetch(first + mine);
  for (int64_t base = first; base < p.n; base += step) {
    const int64_t row = base + mine;
    const bool active = row < p.n;
    Pairs out, b, g;
    float mean = 0.f, inv = 1.f;
    X::values(out, raw_x);
    if (p.block) X::values(b, raw_b);
    if (gated) X::values(g, raw_g);
    const float rg = p.gate && !gated ? sigmoid<T>(Row<T>::get(raw_rg)) : 1.f;
    if (base + step < p.n) fetch(row + step);
    if (p.block) {
      if (p.param[0]) {
        statistics<X, CENTER>(b, red, c, t, p.eps, mean, inv);
#pragma unroll
        for (int k = 0; k < P; ++k) b[k] = mul2(normalised<CENTER>(b[k], mean, inv), weight[k]);
        if (BIAS && p.param[1]) {
          Pairs w;
          X::param(w, p.param[1], p.param_dtype[1], 0.f, c, t, lanes);
#pragma unroll
          for (int k = 0; k < P; ++k) b[k] = add2(b[k], w[k]);
        }
      }
      if (p.stats && t == 0 && active) *(float2*)(p.stats + row * 4) = make_float2(mean, inv);
#pragma unroll
      for (int k = 0; k < P; ++k) out[k] = fma2(mul2(scale[k], gated ? sigmoid<T>(g[k]) : pair(rg)), b[k], out[k]);
      if (p.out) X::store(out, p.out, row, c, t, lanes, active);
    }
    if (p.normed) {
      if (BIAS || CENTER) {                                         // what a bias, or a mean, left behind the row's end
#pragma unroll
        for (int k = 0; k < P; ++k) {
          if (!X::inside(2 * k, c, t, lanes)) out[k].x = 0.f;
          if (!X::inside(2 * k + 1, c, t, lanes)) out[k].y = 0.f;
        }
      }
      statistics<X, CENTER>(out, red, c, t, p.eps, mean, inv);
      if (p.stats && t == 0 && active) *(float2*)(p.stats + row * 4 + 2) = make_float2(mean, inv);
#pragma unroll
      for (int k = 0; k < P; ++k) out[k] = mul2(normalised<CENTER>(out[k], mean, inv), next_weight[k]);
      if (BIAS && p.param[4]) {
        X::param(b, p.param[4], p.param_dtype[4], 0.f, c, t, lanes);
#pragma unroll
        for (int k = 0; k < P; ++k) out[k] = add2(out[k], b[k]);
      }
      X::store(out, p.normed, row, c, t, lanes, active);
    }
  }
}

template <typename T, int VEC, int NV, bool CENTER, bool BIAS, int THREADS>
__global__ void __launch_bounds__(THREADS, backward_blocks_per_sm(THREADS)) backward_kernel(const __grid_constant__ Params p) {
  using X = Tile<T, VEC, NV>;
  constexpr int E = X::E, P = X::P;
  using Pairs = typename X::Pairs;
  __shared__ float slots[2][kMaxWarps][4];
  constexpr bool kWide = E == 16;
  extern __shared__ __align__(16) float columns[];                  // rows of a block > 1: [E][kBlock]; wide: [kSums][P] pairs of THREADS
  after_previous();
  const int lanes = p.lanes, c = p.c, t = threadIdx.x & (lanes - 1), rows = blockDim.x / lanes;
  const bool gated = p.gate && !p.gate_row;
  const float per_c = 1.f / (float)c;
  Reducer red{slots, lanes, 0};
  Pairs weight, scale, next_weight;
  X::param(weight, p.param[0], p.param_dtype[0], 1.f, c, t, lanes);
  X::param(scale, p.param[2], p.param_dtype[2], 1.f, c, t, lanes);
  X::param(next_weight, p.param[3], p.param_dtype[3], 1.f, c, t, lanes);
  float2 in_registers[kWide ? 1 : kSums][kWide ? 1 : P];
  auto sums = [&](int s, int k) -> float2& {
    if constexpr (kWide) return ((float2*)columns)[(s * P + k) * THREADS + threadIdx.x];
    else return in_registers[s][k];
  };
#pragma unroll
  for (int s = 0; s < kSums; ++s)
#pragma unroll
    for (int k = 0; k < P; ++k) sums(s, k) = pair(0.f);
  typename X::Raw raw_x, raw_b, raw_g, raw_d, raw_n;
  typename Row<T>::Bits raw_rg = 0;
  float4 raw_st = make_float4(0.f, 0.f, 0.f, 0.f);
  auto fetch = [&](int64_t row) {
    const bool some = row < p.n;
    raw_st = some ? *(const float4*)(p.stats + row * 4) : make_float4(0.f, 0.f, 0.f, 0.f);
    X::fetch(raw_x, p.residual, row, c, t, lanes, some);
    if (p.block) X::fetch(raw_b, p.block, row, c, t, lanes, some);
    if (gated) X::fetch(raw_g, p.gate, row, c, t, lanes, some);
    else if (p.gate) raw_rg = some ? ((const typename Row<T>::Bits*)p.gate)[row] : (typename Row<T>::Bits)0;
    if (p.d_out) X::fetch(raw_d, p.d_out, row, c, t, lanes, some);
    if (p.d_normed) X::fetch(raw_n, p.d_normed, row, c, t, lanes, some);
  };
  const int64_t first = (int64_t)blockIdx.x * rows, step = (int64_t)gridDim.x * rows;
  const int mine = threadIdx.x / lanes;
  if (!kWide && first < p.n) fetch(first + mine);
  for (int64_t base = first; base < p.n; base += step) {
    const int64_t row = base + mine;
    const bool active = row < p.n;
    Pairs x, b, g, total, dn;
    if (kWide) fetch(row);
    const float4 st = raw_st;
    const float mb = p.param[0] ? st.x : 0.f, ib = p.param[0] ? st.y : 1.f;
    const float rg = p.gate && !gated ? sigmoid<T>(Row<T>::get(raw_rg)) : 1.f;
    X::values(x, raw_x);
    if (p.block) X::values(b, raw_b);
    if (gated) X::values(g, raw_g);
    if (p.d_out) {
      X::values(total, raw_d);
    } else {
#pragma unroll
      for (int k = 0; k < P; ++k) total[k] = pair(0.f);
    }
    if (p.d_normed) X::values(dn, raw_n);
    if (!kWide && base + step < p.n) fetch(row + step);
    Pairs bias;                                                     // in registers only where there is one
    if (BIAS) X::param(bias, p.param[1], p.param_dtype[1], 0.f, c, t, lanes);
    auto inner = [&](int k) { return BIAS ? fma2(b[k], weight[k], bias[k]) : mul2(b[k], weight[k]); };
    if (p.block) {                                                  // b: the normalised block
#pragma unroll
      for (int k = 0; k < P; ++k) {
        b[k] = normalised<CENTER>(b[k], mb, ib);
        g[k] = gated ? sigmoid<T>(g[k]) : pair(rg);
      }
    }
    if (p.d_normed) {
      float2 s0 = pair(0.f), s1 = pair(0.f);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        if (p.block) x[k] = fma2(mul2(scale[k], g[k]), inner(k), x[k]);
        x[k] = normalised<CENTER>(x[k], st.z, st.w);                // the normalised out; dn is zero behind the row
        sums(3, k) = fma2(dn[k], x[k], sums(3, k));
        if (BIAS) sums(4, k) = add2(sums(4, k), dn[k]);
        dn[k] = mul2(dn[k], next_weight[k]);
        s0 = fma2(dn[k], x[k], s0);
        if (CENTER) s1 = add2(s1, dn[k]);
      }
      float s[CENTER ? 2 : 1];
      s[0] = both(s0);
      if (CENTER) s[CENTER] = both(s1);
      red.sum(s);
      const float2 along = pair(-st.w * s[0] * per_c), across = pair(CENTER ? -st.w * s[CENTER] * per_c : 0.f);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        total[k] = fma2(dn[k], pair(st.w), fma2(x[k], along, total[k]));
        if (CENTER) total[k] = add2(total[k], across);
        if (!X::inside(2 * k, c, t, lanes)) total[k].x = 0.f;
        if (!X::inside(2 * k + 1, c, t, lanes)) total[k].y = 0.f;
      }
    }
    if (p.d_residual) X::store(total, p.d_residual, row, c, t, lanes, active);
    if (p.block) {
      float2 s0 = pair(0.f), s1 = pair(0.f), s2 = pair(0.f);
#pragma unroll
      for (int k = 0; k < P; ++k) {
        const float2 in = inner(k), tg = mul2(total[k], g[k]), d_inner = mul2(tg, scale[k]);         // tg: gradient of scale * inner
        sums(2, k) = fma2(tg, in, sums(2, k));
        sums(0, k) = fma2(d_inner, b[k], sums(0, k));
        if (BIAS) sums(1, k) = add2(sums(1, k), d_inner);
        x[k] = mul2(d_inner, in);                                   // gradient of the gate's logit
        x[k] = fma2(mul2(x[k], g[k]), pair(-1.f), x[k]);
        s2 = add2(s2, x[k]);
        dn[k] = mul2(d_inner, weight[k]);
        s0 = fma2(dn[k], b[k], s0);
        if (CENTER) s1 = add2(s1, dn[k]);
      }
      if (gated && p.d_gate) X::store(x, p.d_gate, row, c, t, lanes, active);
      float s[3] = {both(s0), both(s2), CENTER ? both(s1) : 0.f};
      if (CENTER) {
        if (p.param[0] || p.gate_row) red.sum(s);
      } else if (p.gate_row) {
        float u[2] = {s[0], s[1]};
        red.sum(u);
        s[0] = u[0]; s[1] = u[1];
      } else if (p.param[0]) {
        float u[1] = {s[0]};
        red.sum(u);
        s[0] = u[0];
      }
      if (p.gate_row && p.d_gate && t == 0 && active) ((typename Row<T>::Bits*)p.d_gate)[row] = Row<T>::put(s[1]);
      if (p.param[0]) {
        const float2 along = pair(-ib * s[0] * per_c), across = pair(CENTER ? -ib * s[2] * per_c : 0.f);
#pragma unroll
        for (int k = 0; k < P; ++k) {
          dn[k] = fma2(dn[k], pair(ib), mul2(b[k], along));
          if (CENTER) dn[k] = add2(dn[k], across);
        }
      }
      if (p.d_block) X::store(dn, p.d_block, row, c, t, lanes, active);
    }
  }
  // the block's sums over its rows
  if (p.partial == nullptr) return;
#pragma unroll
  for (int s = 0; s < kSums; ++s) {
    if (p.param[s] == nullptr || (!BIAS && (s == 1 || s == 4))) continue;
    float* to = p.partial + ((int64_t)blockIdx.x * kSums + s) * c;
    if (!kWide && rows > 1) {
      __syncthreads();
#pragma unroll
      for (int e = 0; e < E; ++e) columns[e * kBlock + threadIdx.x] = e % 2 ? sums(s, e / 2).y : sums(s, e / 2).x;
      __syncthreads();
      for (int i = threadIdx.x; i < lanes * E; i += blockDim.x) {
        const int e = i / lanes, tt = i - e * lanes;
        const int at = X::column(e / VEC, tt, lanes) + e % VEC;
        if (at < c) {
          float v = 0.f;
          for (int r = 0; r < rows; ++r) v += columns[e * kBlock + r * lanes + tt];
          to[at] = v;
        }
      }
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const int at = X::column(e / VEC, t, lanes) + e % VEC;
        if (at < c) to[at] = e % 2 ? sums(s, e / 2).y : sums(s, e / 2).x;
      }
    }
  }
}

// d_param[s][c] = sum over blocks of partial[block][s][c], in the order of the blocks
struct SumParams {
  const float* partial;
  void* to[kSums];
  int dtype[kSums];
  int blocks, c;
};
__global__ void __launch_bounds__(256) sums_kernel(const __grid_constant__ SumParams p) {
  __shared__ double part[8][32];
  after_previous();
  const int s = blockIdx.y, lane = threadIdx.x & 31, w = threadIdx.x >> 5, col = blockIdx.x * 32 + lane;
  if (p.to[s] == nullptr) return;
  double v = 0.0;
  if (col < p.c)
    for (int b = w; b < p.blocks; b += 8) v += (double)p.partial[((int64_t)b * kSums + s) * p.c + col];
  part[w][lane] = v;
  __syncthreads();
  if (w == 0 && col < p.c) {
    for (int i = 1; i < 8; ++i) v += part[i][lane];
    const float f = (float)v;
    if (p.dtype[s] == SPH_F32) ((float*)p.to[s])[col] = f;
    else if (p.dtype[s] == SPH_F16) ((__half*)p.to[s])[col] = __float2half_rn(f);
    else ((__nv_bfloat16*)p.to[s])[col] = __float2bfloat16_rn(f);
  }
}

struct Shape {
  int vec, nv, lanes, threads;
};

// Threads of a row and pieces a thread holds.  whole: rows are a multiple of 16 bytes, and 16-byte aligned.
bool shape_of(int c, int esize, bool whole, Shape* s) {
  const int full = 16 / esize;
  s->vec = whole ? full : 1;
  // A piece of 16 bytes a thread, or four elements: what backward keeps of a row in registers (float32 rows of 1024 channels, eight values
  // instead of four: backward 97 -> 116 us; bf16 rows of 333, 118 -> 312).  Four values, and eight of 16 bits in a root-mean-square norm
  // without a bias, fit without spilling; eight of 16 bits with a bias or a mean spill 250 to 310 bytes a thread (16384 x 2048 rows, gated:
  // backward 230 us, 120 without), eight of float32 260 to 490, sixteen of either 850 to 1420.  More a thread for rows that would need more
  // than 512 threads, or 256 where the pieces of float32 rows still fit then (2048 channels: forward 74 -> 59 us).
  for (const int e : {4, 8, 16}) {
    if (e < s->vec) continue;
    const int most = e == 4 && s->vec == 4 ? 256 : 512;
    s->nv = e / s->vec;
    s->lanes = 1;
    while (s->lanes < most && s->lanes * e < c) s->lanes *= 2;
    if (s->lanes * e >= c) {
      s->threads = s->lanes > 32 ? s->lanes : kBlock;
      return true;
    }
  }
  return false;
}

int grid_of(const Shape& s, int64_t n, int sms, int per_sm) {
  const int64_t blocks = div_up64(n, s.threads / s.lanes);
  return (int)std::min<int64_t>(blocks, (int64_t)sms * per_sm);
}

bool aligned16(const void* p) { return ((uintptr_t)p & 15) == 0; }
bool params_aligned(const Params& p) {
  for (int s = 0; s < kSums; ++s)
    if (!aligned16(p.param[s])) return false;
  return true;
}

int fill(const sph_norm* a, const char* who, Params* p) {
#define SPH_CHECK_ARG_IN(cond, msg)                                             \
  do {                                                                          \
    if (!(cond)) { set_error("%s: %s", who, msg); return SPH_ERR_INVALID; }     \
  } while (0)
  SPH_CHECK_ARG_IN(a && a->n >= 0 && a->c > 0, "bad sizes");
  SPH_CHECK_ARG_IN(a->dtype == SPH_F32 || a->dtype == SPH_F16 || a->dtype == SPH_BF16, "rows are fp32, fp16 or bf16");
  SPH_CHECK_ARG_IN(a->n == 0 || a->residual, "null pointer");
  SPH_CHECK_ARG_IN(a->block || (!a->gate && !a->param[0] && !a->param[1] && !a->param[2]), "a gate, a scale or a norm of no block");
  SPH_CHECK_ARG_IN(a->param[0] || !a->param[1], "a bias without its weight");
  SPH_CHECK_ARG_IN(a->param[3] || !a->param[4], "a bias without its weight");
  SPH_CHECK_ARG_IN(a->eps >= 0.f, "eps must not be negative or NaN");
  if (a->c > SPH_NORM_MAX_CHANNELS) {
    set_error("%s: %d channels, at most %d are supported", who, a->c, SPH_NORM_MAX_CHANNELS);
    return SPH_ERR_LIMIT;
  }
  for (int s = 0; s < kSums; ++s) {
    SPH_CHECK_ARG_IN(!a->param[s] || a->param_dtype[s] == SPH_F32 || a->param_dtype[s] == SPH_F16 || a->param_dtype[s] == SPH_BF16,
                     "parameters are fp32, fp16 or bf16");
    p->param[s] = a->param[s];
    p->param_dtype[s] = a->param_dtype[s];
  }
#undef SPH_CHECK_ARG_IN
  p->block = a->block; p->residual = a->residual; p->gate = a->gate;
  p->gate_row = a->gate && a->gate_per_row;
  p->n = a->n; p->c = a->c; p->eps = a->eps;
  return SPH_OK;
}

template <typename T, int VEC, int NV, bool CENTER, bool BIAS, int THREADS>
int start(bool backward, int grid, const Shape& s, cudaStream_t st, const Params& p) {
  if (backward) {
    constexpr int E = VEC * NV;
    const auto kernel = backward_kernel<T, VEC, NV, CENTER, BIAS, THREADS>;
    const int smem = E == 16 ? kSums * E * THREADS * 4 : s.threads > s.lanes ? kBlock * E * 4 : 0;
    if (E == 16) SPH_CUDA(allow_smem(kernel, smem));
    launch(kernel, grid, s.threads, smem, st, p);
  } else {
    launch(forward_kernel<T, VEC, NV, CENTER, BIAS, THREADS>, grid, s.threads, 0, st, p);
  }
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}
template <typename T, int VEC, int NV, int THREADS>
int start(bool backward, bool center, int grid, const Shape& s, cudaStream_t st, const Params& p) {
  if (center) return start<T, VEC, NV, true, true, THREADS>(backward, grid, s, st, p);
  if (p.param[1] || p.param[4]) return start<T, VEC, NV, false, true, THREADS>(backward, grid, s, st, p);
  return start<T, VEC, NV, false, false, THREADS>(backward, grid, s, st, p);
}
template <typename T>
int start(bool backward, bool center, int grid, const Shape& s, cudaStream_t st, const Params& p) {
  constexpr int V = Row<T>::kVec;
  const bool large = s.threads > kBlock;
  if (s.vec == 1) {
    if (s.nv == 16) return start<T, 1, 16, 512>(backward, center, grid, s, st, p);
    if (s.nv == 8) return start<T, 1, 8, 512>(backward, center, grid, s, st, p);
    if (large) return start<T, 1, 4, 512>(backward, center, grid, s, st, p);
    return start<T, 1, 4, kBlock>(backward, center, grid, s, st, p);
  }
  if (s.nv == 1 && !large) return start<T, V, 1, kBlock>(backward, center, grid, s, st, p);
  if (s.nv == 2 && large) return start<T, V, 2, 512>(backward, center, grid, s, st, p);
  if constexpr (V == 8) return start<T, V, 1, 512>(backward, center, grid, s, st, p);
  else if (s.nv == 2) return start<T, V, 2, kBlock>(backward, center, grid, s, st, p);
  else return start<T, V, 4, 512>(backward, center, grid, s, st, p);
}
int start(int dtype, bool backward, bool center, int grid, const Shape& s, cudaStream_t st, Params& p) {
  p.lanes = s.lanes;
  if (dtype == SPH_F32) return start<float>(backward, center, grid, s, st, p);
  if (dtype == SPH_F16) return start<__half>(backward, center, grid, s, st, p);
  return start<__nv_bfloat16>(backward, center, grid, s, st, p);
}

}  // namespace

}  // namespace sph

using namespace sph;

extern "C" int sph_residual_norm(const sph_norm* a, void* d_out, void* d_normed, float* d_stats, void* stream) {
  Params p = {};
  const int rc = fill(a, __func__, &p);
  if (rc != SPH_OK) return rc;
  if (a->n == 0) return SPH_OK;
  SPH_CHECK_ARG(!!d_out == !!a->block, "out belongs to a block");
  SPH_CHECK_ARG(!!d_normed == !!a->param[3], "normed belongs to a next_weight");
  SPH_CHECK_ARG(aligned16(d_stats), "the statistics must be 16-byte aligned");
  p.out = d_out; p.normed = d_normed; p.stats = d_stats;
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  const int e = dtype_bytes(a->dtype);
  const bool whole = (int64_t)a->c * e % 16 == 0 && aligned16(a->block) && aligned16(a->residual) &&
                     (p.gate_row || aligned16(a->gate)) && aligned16(d_out) && aligned16(d_normed) && params_aligned(p);
  Shape s;
  if (!shape_of(a->c, e, whole, &s)) { set_error("%s: too many channels", __func__); return SPH_ERR_LIMIT; }
  return start(a->dtype, false, a->center != 0, grid_of(s, a->n, sms, forward_blocks_per_sm(s.threads)), s, (cudaStream_t)stream, p);
}

extern "C" int64_t sph_residual_norm_scratch_bytes(int64_t n, int32_t c) {
  if (n < 0 || c <= 0) { set_error("%s: bad sizes", __func__); return SPH_ERR_INVALID; }
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  int64_t blocks = 1;                         // of any way to read a row
  for (const int way : {0, 1, 2}) {
    Shape s;
    if (!shape_of(c, way == 0 ? 2 : 4, way != 2, &s)) {
      set_error("%s: %d channels, at most %d are supported", __func__, c, SPH_NORM_MAX_CHANNELS);
      return SPH_ERR_LIMIT;
    }
    blocks = std::max<int64_t>(blocks, grid_of(s, n, sms, backward_blocks_per_sm(s.threads)));
  }
  return blocks * kSums * c * (int64_t)sizeof(float);
}

extern "C" int sph_residual_norm_backward(const sph_norm* a, const void* d_dout, const void* d_dnormed, const float* d_stats,
                                          void* d_scratch, void* d_dblock, void* d_dresidual, void* d_dgate, void* const d_dparam[5],
                                          void* stream) {
  Params p = {};
  const int rc = fill(a, __func__, &p);
  if (rc != SPH_OK) return rc;
  SPH_CHECK_ARG(d_dparam, "null pointer");
  SPH_CHECK_ARG(!d_dnormed || a->param[3], "a gradient of normed without a next_weight");
  SPH_CHECK_ARG(!d_dout || a->block, "a gradient of out without a block");
  SPH_CHECK_ARG(a->n == 0 || (d_stats && aligned16(d_stats)), "the statistics must be given, 16-byte aligned");
  SPH_CHECK_ARG(d_scratch, "null scratch");
  for (int s = 0; s < kSums; ++s) SPH_CHECK_ARG(a->param[s] || !d_dparam[s], "a gradient of a parameter that there is not");
  p.d_out = d_dout; p.d_normed = d_dnormed;
  p.d_block = d_dblock; p.d_residual = d_dresidual; p.d_gate = d_dgate;
  p.stats = const_cast<float*>(d_stats);
  p.partial = (float*)d_scratch;
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  const int e = dtype_bytes(a->dtype);
  const bool whole = (int64_t)a->c * e % 16 == 0 && aligned16(a->block) && aligned16(a->residual) &&
                     (p.gate_row || (aligned16(a->gate) && aligned16(d_dgate))) && aligned16(d_dout) && aligned16(d_dnormed) &&
                     aligned16(d_dblock) && aligned16(d_dresidual) && params_aligned(p);
  Shape s;
  if (!shape_of(a->c, e, whole, &s)) { set_error("%s: too many channels", __func__); return SPH_ERR_LIMIT; }
  SumParams q = {};
  q.partial = p.partial;
  q.c = a->c;
  if (a->n > 0) {
    q.blocks = grid_of(s, a->n, sms, backward_blocks_per_sm(s.threads));
    const int done = start(a->dtype, true, a->center != 0, q.blocks, s, (cudaStream_t)stream, p);
    if (done != SPH_OK) return done;
  }
  bool any = false;
  for (int i = 0; i < kSums; ++i) {
    q.to[i] = d_dparam[i];
    q.dtype[i] = a->param_dtype[i];
    any |= d_dparam[i] != nullptr;
  }
  if (any) {
    launch(sums_kernel, dim3(div_up(a->c, 32), kSums), 256, 0, (cudaStream_t)stream, q);
    SPH_LAUNCH_CHECK();
  }
  return SPH_OK;
}
