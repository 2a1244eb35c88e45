// Cross attention of queries to the rows of their scan: the kernels on the CUDA cores, for float32 and for rows that the tensor-core
// kernels do not take, the sums over parts that both kinds leave, and the entry points.
//
//   S = scale Q K^T, masked keys -inf;  P = softmax of its rows;  O = P V
//   delta = rowsum(dO O);  dP = dO V^T;  dS = P (dP - delta);  dQ = scale dS K;  dK = scale dS^T Q;  dV = P^T dO
//
// A block has a tile of 64 rows and walks the other side in tiles of 64: forward with the running maximum and sum of a softmax, backward
// with the logarithm of the sum from the forward pass, once for queries (dQ) and once for keys (dK and dV), so that nothing is added
// atomically and results are the same every time.  256 threads hold 4 x 4 scores each.  The longer side is split over blocks where
// the tiles do not fill the GPU; each leaves its part in float32, and a launch more joins them in their order.
//
// Rows that are no keys are read as zeros: what they hold does not matter, NaN included.  A query without keys has zeros.
#include <algorithm>
#include <type_traits>

#include "attention.cuh"

namespace sph {

namespace attn {

constexpr int kTile = 64;
constexpr int kThreads = 256;
constexpr int kScorePitch = kTile + 4;
constexpr int kTcTile = 128, kTcStep = 64;    // rows of a tile and of a step of its walk in the tensor-core kernels
constexpr int kMostParts = 64;                // of a walk: two lanes of a warp have them all

template <typename T> __device__ __forceinline__ float to_float(T v);
template <> __device__ __forceinline__ float to_float(float v) { return v; }
template <> __device__ __forceinline__ float to_float(__half v) { return __half2float(v); }
template <> __device__ __forceinline__ float to_float(__nv_bfloat16 v) { return __bfloat162float(v); }
template <typename T> __device__ __forceinline__ T from_float(float v);
template <> __device__ __forceinline__ float from_float(float v) { return v; }
template <> __device__ __forceinline__ __half from_float(float v) { return __float2half_rn(v); }
template <> __device__ __forceinline__ __nv_bfloat16 from_float(float v) { return __float2bfloat16_rn(v); }

// 64 rows of d elements to shared memory as float32, zeros where there is no row (row(r) is null) and behind d.
template <typename T, int DP, typename Row>
__device__ __forceinline__ void load_tile(float* to, int d, int vec, Row row) {
  constexpr int PITCH = DP + 4;
  constexpr int E = 16 / sizeof(T);
  if (vec) {
    for (int i = threadIdx.x; i < kTile * (DP / E); i += kThreads) {
      const int r = i / (DP / E), c = i % (DP / E) * E;
      const T* src = row(r);
      struct __align__(16) Piece { T v[E]; } piece;
      const bool some = src != nullptr && c < d;
      if (some) piece = *(const Piece*)(src + c);
#pragma unroll
      for (int j = 0; j < E; j += 4)
        *(float4*)(to + r * PITCH + c + j) = some ? make_float4(to_float(piece.v[j]), to_float(piece.v[j + 1]), to_float(piece.v[j + 2]),
                                                                to_float(piece.v[j + 3]))
                                                  : make_float4(0.f, 0.f, 0.f, 0.f);
    }
  } else {
    for (int i = threadIdx.x; i < kTile * DP; i += kThreads) {
      const int r = i / DP, c = i % DP;
      const T* src = row(r);
      to[r * PITCH + c] = src != nullptr && c < d ? to_float(src[c]) : 0.f;
    }
  }
}

// s[i][j] = a[4 ty + i] . b[tx + 16 j], even and odd channels apart: two to an operation
template <int DP>
__device__ __forceinline__ void scores(float (&s)[4][4], const float* a, const float* b, int d, int tx, int ty) {
  constexpr int PITCH = DP + 4;
  float2 sum[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) sum[i][j] = make_float2(0.f, 0.f);
#pragma unroll 2
  for (int c = 0; c < d; c += 4) {            // zeros up to a multiple of 4
    float4 x[4], y[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = *(const float4*)(a + (4 * ty + i) * PITCH + c);
#pragma unroll
    for (int j = 0; j < 4; ++j) y[j] = *(const float4*)(b + (tx + 16 * j) * PITCH + c);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        sum[i][j] = fma2(make_float2(x[i].x, x[i].y), make_float2(y[j].x, y[j].y), sum[i][j]);
        sum[i][j] = fma2(make_float2(x[i].z, x[i].w), make_float2(y[j].z, y[j].w), sum[i][j]);
      }
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) s[i][j] = sum[i][j].x + sum[i][j].y;
}

// A thread's channels of a row: pieces of W consecutive ones, piece j at 16 W j + W tx.
template <int DP>
struct Columns {
  static constexpr int W = DP >= 64 ? 4 : 2, N = DP / 16 / W;
};

// acc[i] += sum over n of p[4 ty + i][n] * v[n], channels two to an operation
template <int DP>
__device__ __forceinline__ void accumulate(float2 (&acc)[4][DP / 32], const float* p, const float* v, int tx, int ty) {
  constexpr int PITCH = DP + 4, W = Columns<DP>::W, N = Columns<DP>::N;
#pragma unroll 2
  for (int n = 0; n < kTile; n += 4) {
    float x[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const float4 f = *(const float4*)(p + (4 * ty + i) * kScorePitch + n);
      x[i][0] = f.x; x[i][1] = f.y; x[i][2] = f.z; x[i][3] = f.w;
    }
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int j = 0; j < N; ++j) {
        float2 y[W / 2];
        const float* from = v + (n + m) * PITCH + 16 * W * j + W * tx;
        if constexpr (W == 4) {
          const float4 f = *(const float4*)from;
          y[0] = make_float2(f.x, f.y);
          y[1] = make_float2(f.z, f.w);
        } else {
          y[0] = *(const float2*)from;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
          for (int w = 0; w < W / 2; ++w)
            acc[i][j * W / 2 + w] = fma2(make_float2(x[i][m], x[i][m]), y[w], acc[i][j * W / 2 + w]);
      }
  }
}

template <typename T, int DP>
__device__ __forceinline__ void store_row(const float2 (&acc)[DP / 32], float by, T* to, int d, int tx) {
  constexpr int W = Columns<DP>::W, N = Columns<DP>::N;
#pragma unroll
  for (int j = 0; j < N; ++j)
#pragma unroll
    for (int w = 0; w < W; ++w) {
      const int c = 16 * W * j + W * tx + w;
      const float2 pair = acc[(j * W + w) / 2];
      if (c < d) to[c] = from_float<T>((w % 2 ? pair.y : pair.x) * by);
    }
}

template <bool QUERIES>
__device__ __forceinline__ Work block_work(const Params& p) {
  __shared__ Work s_work;
  if (threadIdx.x < 32) {
    const Work w = find_work<QUERIES>(p, blockIdx.x / p.hkv, kTile, kTile);
    if (threadIdx.x == 0) s_work = w;
  }
  __syncthreads();
  return s_work;
}

template <typename T, int DP>
__global__ void __launch_bounds__(kThreads) forward_kernel(const __grid_constant__ Params p) {
  constexpr int PITCH = DP + 4;
  extern __shared__ __align__(16) float smem[];
  float *s_q = smem, *s_k = s_q + kTile * PITCH, *s_v = s_k + kTile * PITCH, *s_p = s_v + kTile * PITCH;
  __shared__ uint8_t s_key[kTile];
  after_previous();
  report_scans(p);
  const int key_head = blockIdx.x % p.hkv;
  const Work w = block_work<true>(p);
  if (w.scan < 0) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int rows = min(kTile, w.nq * p.group - w.tile * kTile);       // of the tile
  auto query = [&](int r, int* head) {
    const int i = w.tile * kTile + r;
    *head = key_head * p.group + i % p.group;
    return w.q0 + i / p.group;
  };
  load_tile<T, DP>(s_q, p.d, p.vec, [&](int r) -> const T* {
    int h;
    const int64_t q = query(min(r, rows - 1), &h);
    return r < rows ? (const T*)p.q + q * p.q_row + h * p.q_head : nullptr;
  });
  const int2 keys = make_int2(w.first, w.last);
  float2 o[4][DP / 32];
  float top[4], sum[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    top[i] = -INFINITY;
    sum[i] = 0.f;
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) o[i][j] = make_float2(0.f, 0.f);
  }
  for (int k0 = keys.x; k0 < keys.y; k0 += kTile) {
    __syncthreads();
    if (threadIdx.x < kTile) {
      const int k = k0 + threadIdx.x;
      s_key[threadIdx.x] = k < keys.y && (p.mask == nullptr || p.mask[w.k0 + k] != 0);
    }
    __syncthreads();
    load_tile<T, DP>(s_k, p.d, p.vec, [&](int r) -> const T* {
      return s_key[r] ? (const T*)p.k + (int64_t)(w.k0 + k0 + r) * p.k_row + key_head * p.k_head : nullptr;
    });
    load_tile<T, DP>(s_v, p.d, p.vec, [&](int r) -> const T* {
      return s_key[r] ? (const T*)p.v + (int64_t)(w.k0 + k0 + r) * p.v_row + key_head * p.v_head : nullptr;
    });
    __syncthreads();
    float s[4][4];
    scores<DP>(s, s_q, s_k, p.d, tx, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      float most = -INFINITY;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = s_key[tx + 16 * j] ? s[i][j] * p.scale_log2 : -INFINITY;
        most = fmaxf(most, s[i][j]);
      }
#pragma unroll
      for (int of = 8; of > 0; of >>= 1) most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, of));
      const float now = fmaxf(top[i], most);
      const float base = now == -INFINITY ? 0.f : now;                // nothing yet: every 2^(-inf - 0) is zero
      const float by = exp2f(top[i] - base);
      top[i] = now;
      float add = 0.f;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = exp2f(s[i][j] - base);
        add += s[i][j];
        s_p[(4 * ty + i) * kScorePitch + tx + 16 * j] = s[i][j];
      }
      sum[i] = sum[i] * by + add;                                     // of this thread's columns; joined at the end
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) o[i][j] = mul2(o[i][j], make_float2(by, by));
    }
    __syncwarp();                                                     // a row of P belongs to half a warp
    accumulate<DP>(o, s_p, s_v, tx, ty);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
#pragma unroll
    for (int of = 8; of > 0; of >>= 1) sum[i] += __shfl_xor_sync(0xffffffffu, sum[i], of);
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    int h;
    const int64_t q = query(r, &h);
    const bool none = sum[i] == 0.f;
    const float by = none ? 0.f : 1.f / sum[i], lse = none ? INFINITY : top[i] + log2f(sum[i]);
    if (p.parts > 1) {
      const int64_t at = ((int64_t)w.part * p.n_q + q) * p.hq + h;
      store_row<float, DP>(o[i], by, p.part + at * p.d, p.d, tx);
      if (tx == 0) p.part_lse[at] = lse;
      if (tx == 0 && w.part == 0) p.part_count[at] = w.parts;
    } else {
      store_row<T, DP>(o[i], by, (T*)p.out + (q * p.hq + h) * p.d, p.d, tx);
      if (tx == 0 && p.lse) p.lse[q * p.hq + h] = lse;
    }
  }
}

// KEYS: a tile of keys against all queries of the scan (dK, dV); else a tile of queries against its keys (dQ).
template <typename T, int DP, bool KEYS>
__global__ void __launch_bounds__(kThreads) backward_kernel(const __grid_constant__ Params p) {
  constexpr int PITCH = DP + 4;
  extern __shared__ __align__(16) float smem[];
  float *s_r1 = smem, *s_r2 = s_r1 + kTile * PITCH;                   // rows: K and V, or Q and dO
  float *s_c1 = s_r2 + kTile * PITCH, *s_c2 = s_c1 + kTile * PITCH;   // columns: Q and dO, or K and V
  float *s_ds = s_c2 + kTile * PITCH, *s_p = s_ds + kTile * kScorePitch;
  __shared__ float s_lse[kTile], s_delta[kTile];
  __shared__ uint8_t s_key[kTile];
  after_previous();
  const int key_head = blockIdx.x % p.hkv;
  const Work w = block_work<!KEYS>(p);
  if (w.scan < 0) return;
  const int tx = threadIdx.x & 15, ty = threadIdx.x >> 4;
  const int all = w.nq * p.group;
  auto query = [&](int i, int* head) {                                // row i of the scan's queries
    *head = key_head * p.group + i % p.group;
    return (int64_t)w.q0 + i / p.group;
  };
  auto load_queries = [&](float* q_to, float* d_to, int first, int n) {
    load_tile<T, DP>(q_to, p.d, p.vec, [&](int r) -> const T* {
      if (r >= n) return nullptr;
      int h;
      const int64_t q = query(first + r, &h);
      return (const T*)p.q + q * p.q_row + h * p.q_head;
    });
    load_tile<T, DP>(d_to, p.d, p.vec, [&](int r) -> const T* {
      if (r >= n) return nullptr;
      int h;
      const int64_t q = query(first + r, &h);
      return (const T*)p.d_out + (q * p.hq + h) * p.d;
    });
    if (threadIdx.x < kTile) {
      float lse = INFINITY, delta = 0.f;
      if ((int)threadIdx.x < n) {
        int h;
        const int64_t q = query(first + threadIdx.x, &h);
        lse = p.lse[q * p.hq + h];
        delta = p.delta[q * p.hq + h];
      }
      s_lse[threadIdx.x] = lse;
      s_delta[threadIdx.x] = delta;
    }
  };
  auto load_keys = [&](float* k_to, float* v_to, int first, int n) {  // between two barriers of their own
    if (threadIdx.x < kTile)
      s_key[threadIdx.x] = (int)threadIdx.x < n && (p.mask == nullptr || p.mask[w.k0 + first + threadIdx.x] != 0);
    __syncthreads();
    load_tile<T, DP>(k_to, p.d, p.vec, [&](int r) -> const T* {
      return s_key[r] ? (const T*)p.k + (int64_t)(w.k0 + first + r) * p.k_row + key_head * p.k_head : nullptr;
    });
    load_tile<T, DP>(v_to, p.d, p.vec, [&](int r) -> const T* {
      return s_key[r] ? (const T*)p.v + (int64_t)(w.k0 + first + r) * p.v_row + key_head * p.v_head : nullptr;
    });
  };
  const int row0 = w.tile * kTile, rows = min(kTile, (KEYS ? w.nk : all) - row0);
  if (KEYS) load_keys(s_r1, s_r2, row0, rows);
  else load_queries(s_r1, s_r2, row0, rows);
  const int2 span = make_int2(w.first, w.last);
  float2 a1[4][DP / 32], a2[4][DP / 32];                              // dV ; dK or dQ
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < DP / 32; ++j) a1[i][j] = a2[i][j] = make_float2(0.f, 0.f);
  for (int c0 = span.x; c0 < span.y; c0 += kTile) {
    __syncthreads();
    if (KEYS) load_queries(s_c1, s_c2, c0, min(kTile, span.y - c0));
    else load_keys(s_c1, s_c2, c0, min(kTile, span.y - c0));
    __syncthreads();
    float s[4][4], t[4][4];
    scores<DP>(s, s_r1, s_c1, p.d, tx, ty);
    scores<DP>(t, s_r2, s_c2, p.d, tx, ty);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = 4 * ty + i, c = tx + 16 * j, q = KEYS ? c : r, k = KEYS ? r : c;
        const float x = s_key[k] ? exp2f(fmaf(s[i][j], p.scale_log2, -s_lse[q])) : 0.f;
        if (KEYS) s_p[r * kScorePitch + c] = x;
        s_ds[r * kScorePitch + c] = x * (t[i][j] - s_delta[q]);
      }
    __syncwarp();
    if (KEYS) accumulate<DP>(a1, s_p, s_c2, tx, ty);
    accumulate<DP>(a2, s_ds, s_c1, tx, ty);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int r = 4 * ty + i;
    if (r >= rows) continue;
    if (KEYS ? !s_key[r] : s_lse[r] == INFINITY) {                    // no key, or a query without: zeros, whatever the other side holds
#pragma unroll
      for (int j = 0; j < DP / 32; ++j) a1[i][j] = a2[i][j] = make_float2(0.f, 0.f);
    }
    int64_t at_row;                                                   // of [rows][heads]
    if (KEYS) {
      at_row = (int64_t)(w.k0 + row0 + r) * p.hkv + key_head;
    } else {
      int h;
      const int64_t q = query(row0 + r, &h);
      at_row = q * p.hq + h;
    }
    if (p.parts > 1) {
      if (tx == 0 && w.part == 0) p.part_count[at_row] = w.parts;
      at_row += (int64_t)w.part * (KEYS ? (int64_t)p.n_k * p.hkv : (int64_t)p.n_q * p.hq);
      store_row<float, DP>(a2[i], p.scale, p.part + at_row * p.d, p.d, tx);
      if (KEYS) store_row<float, DP>(a1[i], 1.f, p.part2 + at_row * p.d, p.d, tx);
    } else {
      store_row<T, DP>(a2[i], p.scale, (T*)(KEYS ? p.dk : p.dq) + at_row * p.d, p.d, tx);
      if (KEYS) store_row<T, DP>(a1[i], 1.f, (T*)p.dv + at_row * p.d, p.d, tx);
    }
  }
}

// delta of every row of every query head, a warp each; with dq.plan the first two warps plan what the tensor-core kernels do, for dQ and
// for dK and dV.
template <typename T>
__global__ void __launch_bounds__(kThreads) delta_kernel(const T* d_out, const T* out, float* delta, int64_t rows, int d,
                                                         const __grid_constant__ Params dq, const __grid_constant__ Params dkv) {
  after_previous();
  const int lane = threadIdx.x & 31;
  if (dq.plan != nullptr && blockIdx.x == 0 && threadIdx.x < 64) {
    const Params& p = threadIdx.x < 32 ? dq : dkv;
    auto leave = [&](const ScanPlan& x, int s0) {
      if (s0 + lane < p.B + 2) const_cast<ScanPlan*>(p.plan)[s0 + lane] = x;
      return false;
    };
    if (threadIdx.x < 32) plan_scans<true>(p, kTcTile, kTcStep, leave);
    else plan_scans<false>(p, kTcTile, kTcStep, leave);
  }
  for (int64_t r = (int64_t)blockIdx.x * (kThreads / 32) + (threadIdx.x >> 5); r < rows; r += (int64_t)gridDim.x * (kThreads / 32)) {
    float s = 0.f;
    for (int c = lane; c < d; c += 32) s = fmaf(to_float(d_out[r * d + c]), to_float(out[r * d + c]), s);
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    if (lane == 0) delta[r] = s;
  }
}

// Parts of the forward pass: out = sum of 2^(lse_i - lse) part_i with lse = log2 of the sum of 2^lse_i.  WARPS warps a row, that share the
// parts; of a warp, lanes the parts' lse first, then the channels.
template <typename T, int WARPS>
__global__ void __launch_bounds__(kThreads) join_forward_kernel(const float* part, const float* part_lse, const int* count, int most,
                                                                int64_t rows, int d, T* out, float* lse) {
  constexpr int kRows = kThreads / 32 / WARPS;              // of a block
  __shared__ float s_v[kThreads / 32][SPH_ATTENTION_MAX_CHANNELS];
  after_previous();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  for (int64_t r0 = (int64_t)blockIdx.x * kRows; r0 < rows; r0 += (int64_t)gridDim.x * kRows) {
    const int64_t r = r0 + warp / WARPS;
    const bool mine = r < rows;
    const int splits = mine ? min(max(count[r], 0), most) : 0;        // unordered scans may have left it unwritten
    float l[2];                                             // of parts lane and lane + 32; +inf: one without keys
    float top = -INFINITY;
    bool some = false;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      const int s = lane + 32 * i;
      l[i] = mine && s < splits ? part_lse[(int64_t)s * rows + r] : INFINITY;
      some |= l[i] != INFINITY;
      top = fmaxf(top, l[i] == INFINITY ? -INFINITY : l[i]);          // NaN is left to the sum
    }
    for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    some = __any_sync(0xffffffffu, some);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
      l[i] = l[i] == INFINITY ? 0.f : exp2f(l[i] - base);   // weights from here on
      sum += l[i];
    }
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    const float inv = some ? 1.f / sum : 0.f;
    float v[SPH_ATTENTION_MAX_CHANNELS / 32] = {0.f, 0.f, 0.f, 0.f};
    for (int s = warp % WARPS; s < splits; s += WARPS) {    // a warp has one row
      const float f = __shfl_sync(0xffffffffu, s < 32 ? l[0] : l[1], s & 31) * inv;
      if (f == 0.f) continue;                               // a part without keys is not looked at
#pragma unroll
      for (int i = 0; i < SPH_ATTENTION_MAX_CHANNELS / 32; ++i)
        if (lane + 32 * i < d) v[i] = fmaf(f, part[((int64_t)s * rows + r) * d + lane + 32 * i], v[i]);
    }
    if (WARPS > 1) {
#pragma unroll
      for (int i = 0; i < SPH_ATTENTION_MAX_CHANNELS / 32; ++i) s_v[warp][lane + 32 * i] = v[i];
      __syncthreads();
      if (warp % WARPS == 0) {
#pragma unroll
        for (int i = 0; i < SPH_ATTENTION_MAX_CHANNELS / 32; ++i)
          for (int x = 1; x < WARPS; ++x) v[i] += s_v[warp + x][lane + 32 * i];
      }
      __syncthreads();
    }
    if (mine && warp % WARPS == 0) {
#pragma unroll
      for (int i = 0; i < SPH_ATTENTION_MAX_CHANNELS / 32; ++i)
        if (lane + 32 * i < d) out[r * d + lane + 32 * i] = from_float<T>(v[i]);
      if (lane == 0 && lse) lse[r] = some ? base + log2f(sum) : INFINITY;
    }
  }
}

// Parts of a gradient, added in their order.
template <typename T>
__global__ void __launch_bounds__(kThreads) join_sum_kernel(const float* part, const int* count, int most, int64_t n, int d, T* to) {
  after_previous();
  for (int64_t i = (int64_t)blockIdx.x * kThreads + threadIdx.x; i < n; i += (int64_t)gridDim.x * kThreads) {
    const int parts = min(max(count[i / d], 0), most);
    float v = 0.f;
    for (int s = 0; s < parts; ++s) v += part[(int64_t)s * n + i];
    to[i] = from_float<T>(v);
  }
}

int attention_forward_tc(const Params& p, bool bf16, int blocks, cudaStream_t st);      // attention_tc.cu
// attention_decode.cu
int attention_decode_rows(int dtype, int64_t rows);
int attention_decode(const Params& p, int dtype, int rows, int blocks, cudaStream_t st);
// attention_tc_bwd.cu
int attention_backward_tc(const Params& p, bool bf16, bool keys, int blocks, cudaStream_t st);

namespace {

// 16-bit rows in pieces of 16 bytes go to the tensor cores; there the largest score is found before it is scaled, so not with a
// scale that is negative or zero.
bool on_tensor_cores(const sph_attention& a, const Params& p) {
  return (a.dtype == SPH_F16 || a.dtype == SPH_BF16) && p.vec && p.scale > 0.f;
}

int padded(int d) { return d <= 32 ? 32 : d <= 64 ? 64 : 128; }
int forward_smem(int dp) { return (3 * kTile * (dp + 4) + kTile * kScorePitch) * 4; }
int backward_smem(int dp, bool keys) { return (4 * kTile * (dp + 4) + (keys ? 2 : 1) * kTile * kScorePitch) * 4; }

// Parts that the walk of `blocks` blocks over `tiles` tiles each is split into on average, where `slots` blocks run at a time.  What it
// costs, in tiles' time: the rounds of parts that there are, as whole ones and as they would be if every slot went on at once, taken by
// half (the device makes the parts of scans of different length equally long, but not their number a multiple of the slots), `start` for a
// block to start; and writing and reading parts of `values`, of which `rate` are a tile's time.
int splits_for(int64_t blocks, int64_t slots, int64_t tiles, int64_t values, double start, double rate) {
  int best = 1;
  double least = 1e300;
  for (int64_t s = 1; s <= std::min<int64_t>(kMostParts, std::max<int64_t>(1, tiles / 2)); ++s) {
    const double part = (double)tiles / s + start;
    const double rounds = 0.5 * (double)div_up64(blocks * s, slots) + 0.5 * (std::max(1.0, (double)(blocks * s) / slots) + 0.25);
    const double cost = rounds * part + (s > 1 ? start + s * (double)values / rate : 0.0);
    if (cost < least) { least = cost; best = (int)s; }
  }
  return best;
}

// Of a direction: parts of a tile's walk, at most, and blocks.
struct Split {
  int parts, aim, items;                     // items: what a head's part of the grid has room for
};
struct Plan {
  int decode;                                // rows of a block of the decoding kernel; 0: another one runs forward
  Split fwd, dq, dkv;
};
Plan plan_of(const sph_attention& a, const Params& params, int sms) {
  const int group = a.q_heads / a.k_heads, dp = padded(a.channels);
  const int64_t room = 227 * 1024;
  auto per_sm = [&](int smem) { return std::min<int64_t>(room / (smem + 1024), 4); };
  Plan p;
  const int64_t B = std::max(a.B, 1);
  const int64_t q_rows = a.n_q * group, q_values = a.n_q * a.q_heads * a.channels, k_values = 2 * a.n_k * a.k_heads * a.channels;
  // rows in tiles of `size` (a key head's), that walk over `walk` rows in steps of `step`
  auto split = [&](int64_t rows, int64_t size, int64_t walk, int64_t step, int64_t slots, int64_t values, double start, double rate) {
    const int64_t tiles = std::max<int64_t>(1, div_up64(rows, size * B)) * B;             // if scans are of like length
    const int n = splits_for(tiles * a.k_heads, slots, div_up64(walk, B * step), values, start, rate);
    const int64_t most = most_tiles(rows, size, a.B);
    // of scans that are longer than the others a tile has more parts
    return n == 1 ? Split{1, 1, (int)most} : Split{std::min(4 * n, kMostParts), (int)(tiles * n), (int)(most + tiles * n)};
  };
  if (on_tensor_cores(a, params)) {          // 0.7 us a tile; a block starts in 5 us, one that takes several tiles of rows in 2
    constexpr double kRate = 500000;
    p.fwd = split(q_rows, kTcTile, a.n_k, kTcStep, 2 * sms, q_values, 8, kRate);
    p.dq = split(q_rows, kTcTile, a.n_k, kTcStep, sms, q_values, 4, kRate);
    p.dkv = split(a.n_k, kTcTile, q_rows, kTcStep, sms, k_values, 4, kRate);
  } else {                                   // 4 us a tile
    constexpr double kRate = 3000000;
    p.fwd = split(q_rows, kTile, a.n_k, kTile, sms * per_sm(forward_smem(dp)), q_values, 1, kRate);
    p.dq = split(q_rows, kTile, a.n_k, kTile, sms * per_sm(backward_smem(dp, false)), q_values, 1, kRate);
    p.dkv = split(a.n_k, kTile, q_rows, kTile, sms * per_sm(backward_smem(dp, true)), k_values, 1, kRate);
  }
  p.decode = params.vec ? attention_decode_rows(a.dtype, div_up64(q_rows, B)) : 0;
  if (p.decode) p.fwd = split(q_rows, p.decode, a.n_k, 64, 2 * sms, q_values, 1.5, 500000);
  return p;
}

template <typename K>
int run_kernel(K* kernel, int blocks, int smem, cudaStream_t st, const Params& p) {
  SPH_CUDA(allow_smem(kernel, 227 * 1024 - 2048));
  launch(kernel, blocks, kThreads, smem, st, p);
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}

template <typename T>
int forward(const Params& p, int blocks, cudaStream_t st) {
  const int dp = padded(p.d), smem = forward_smem(dp);
  if (dp == 32) return run_kernel(forward_kernel<T, 32>, blocks, smem, st, p);
  if (dp == 64) return run_kernel(forward_kernel<T, 64>, blocks, smem, st, p);
  return run_kernel(forward_kernel<T, 128>, blocks, smem, st, p);
}
template <typename T, bool KEYS>
int backward(const Params& p, int blocks, cudaStream_t st) {
  const int dp = padded(p.d), smem = backward_smem(dp, KEYS);
  if (dp == 32) return run_kernel(backward_kernel<T, 32, KEYS>, blocks, smem, st, p);
  if (dp == 64) return run_kernel(backward_kernel<T, 64, KEYS>, blocks, smem, st, p);
  return run_kernel(backward_kernel<T, 128, KEYS>, blocks, smem, st, p);
}

unsigned grid_for(int64_t items, int64_t per_block) { return (unsigned)std::min<int64_t>(div_up64(items, per_block), 148 * 16); }

template <typename T>
int run_forward(Params p, const Plan& plan, bool tensor_cores, void* scratch, cudaStream_t st) {
  const int64_t rows = (int64_t)p.n_q * p.hq;
  p.parts = plan.fwd.parts;
  p.aim = plan.fwd.aim;
  if (p.parts > 1) {
    p.part = (float*)scratch;
    p.part_lse = p.part + rows * p.d * p.parts;
    p.part_count = (int*)(p.part_lse + rows * p.parts);
  }
  constexpr int dtype = std::is_same<T, float>::value ? SPH_F32 : std::is_same<T, __half>::value ? SPH_F16 : SPH_BF16;
  const int blocks = plan.fwd.items * p.hkv;
  const int rc = plan.decode    ? attention_decode(p, dtype, plan.decode, blocks, st)
                 : tensor_cores ? attention_forward_tc(p, dtype == SPH_BF16, blocks, st)
                                : forward<T>(p, blocks, st);
  if (rc != SPH_OK || p.parts == 1) return rc;
  // a few rows leave most of the GPU to the parts of a row
  constexpr int kWarps = kThreads / 32;
  auto join = [&](auto* kernel, unsigned grid) {
    launch(kernel, grid, kThreads, 0, st, p.part, p.part_lse, p.part_count, p.parts, rows, p.d, (T*)p.out, p.lse);
  };
  if (rows <= 148 * 4) join(join_forward_kernel<T, kWarps>, grid_for(rows, 1));
  else join(join_forward_kernel<T, 1>, grid_for(rows, kWarps));
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}

template <typename T>
int run_backward(Params p, const Plan& plan, bool tensor_cores, const void* out, void* scratch, cudaStream_t st) {
  constexpr bool bf16 = std::is_same<T, __nv_bfloat16>::value;
  const int64_t rows = (int64_t)p.n_q * p.hq, k_values = (int64_t)p.n_k * p.hkv * p.d;
  float* delta = (float*)scratch;
  p.delta = delta;
  ScanPlan* plans = (ScanPlan*)(delta + (rows + 3) / 4 * 4);
  p.part_count = (int*)(plans + 2 * (p.B + 2));
  p.part = (float*)p.part_count + (std::max(rows, (int64_t)p.n_k * p.hkv) + 3) / 4 * 4;
  Params dq = p, dkv = p;
  dq.parts = plan.dq.parts; dq.aim = plan.dq.aim; dq.plan = tensor_cores ? plans : nullptr;
  dkv.parts = plan.dkv.parts; dkv.aim = plan.dkv.aim; dkv.plan = plans + p.B + 2;
  dkv.part2 = dkv.part + k_values * dkv.parts;
  launch(delta_kernel<T>, std::max(1u, grid_for(rows, kThreads / 32)), kThreads, 0, st, (const T*)p.d_out, (const T*)out, delta, rows, p.d, dq, dkv);
  SPH_LAUNCH_CHECK();
  auto join = [&](const float* part, int parts, int64_t n, void* to) {
    launch(join_sum_kernel<T>, grid_for(n, kThreads), kThreads, 0, st, part, p.part_count, parts, n, p.d, (T*)to);
    SPH_LAUNCH_CHECK();
    return SPH_OK;
  };
  if (p.dq && rows) {
    const int blocks = plan.dq.items * p.hkv;
    int rc = tensor_cores ? attention_backward_tc(dq, bf16, false, blocks, st) : backward<T, false>(dq, blocks, st);
    if (rc == SPH_OK && dq.parts > 1) rc = join(dq.part, dq.parts, rows * p.d, p.dq);
    if (rc != SPH_OK) return rc;
  }
  if ((p.dk || p.dv) && k_values) {
    const int blocks = plan.dkv.items * p.hkv;
    int rc = tensor_cores ? attention_backward_tc(dkv, bf16, true, blocks, st) : backward<T, true>(dkv, blocks, st);
    if (rc == SPH_OK && dkv.parts > 1) rc = join(dkv.part, dkv.parts, k_values, p.dk);
    if (rc == SPH_OK && dkv.parts > 1) rc = join(dkv.part2, dkv.parts, k_values, p.dv);
    if (rc != SPH_OK) return rc;
  }
  return SPH_OK;
}

bool aligned(const void* p, int64_t row, int64_t head, int esize) {
  return ((uintptr_t)p & 15) == 0 && row * esize % 16 == 0 && head * esize % 16 == 0;
}

int fill(const sph_attention* a, const char* who, Params* p) {
  auto bad = [&](const char* what) { set_error("%s: %s", who, what); return SPH_ERR_INVALID; };
  if (!a || a->B < 0 || a->n_q < 0 || a->n_k < 0 || a->q_heads < 1 || a->k_heads < 1 || a->channels < 1) return bad("bad sizes");
  if (a->q_heads % a->k_heads != 0) return bad("query heads must be a multiple of key heads");
  if (a->dtype != SPH_F32 && a->dtype != SPH_F16 && a->dtype != SPH_BF16) return bad("rows are fp32, fp16 or bf16");
  if ((a->n_q > 0 && !a->q) || (a->n_k > 0 && (!a->k || !a->v)) || !a->q_ptr || !a->k_ptr) return bad("null pointer");
  if (!(a->scale == a->scale)) return bad("the scale is NaN");
  if (a->channels > SPH_ATTENTION_MAX_CHANNELS) {
    set_error("%s: %d channels a head, at most %d are supported", who, a->channels, SPH_ATTENTION_MAX_CHANNELS);
    return SPH_ERR_LIMIT;
  }
  // tiles, times their parts, and the rows of a scan (queries times heads) are numbered in 31 bits
  const int64_t most = (int64_t)1 << 29;
  if (a->n_k > most || a->n_q * (a->q_heads / a->k_heads) > most || (a->n_q * a->q_heads / kTile + (a->B + 2ll) * a->k_heads) * 64 > most ||
      (a->n_k * a->k_heads / kTile + (a->B + 2ll) * a->k_heads) * 64 > most) {
    set_error("%s: too many rows", who);
    return SPH_ERR_LIMIT;
  }
  *p = Params{};
  p->q = a->q; p->k = a->k; p->v = a->v;
  p->q_row = a->q_row; p->q_head = a->q_head; p->k_row = a->k_row; p->k_head = a->k_head; p->v_row = a->v_row; p->v_head = a->v_head;
  p->q_ptr = a->q_ptr; p->k_ptr = a->k_ptr; p->mask = a->key_mask;
  p->n_q = (int)a->n_q; p->n_k = (int)a->n_k; p->B = a->B; p->hq = a->q_heads; p->hkv = a->k_heads; p->group = a->q_heads / a->k_heads;
  p->d = a->channels;
  p->scale = a->scale;
  p->scale_log2 = a->scale * kLog2e;
  const int e = dtype_bytes(a->dtype);
  p->vec = (int64_t)p->d * e % 16 == 0 && aligned(p->q, p->q_row, p->q_head, e) && aligned(p->k, p->k_row, p->k_head, e) &&
           aligned(p->v, p->v_row, p->v_head, e);
  return SPH_OK;
}

}  // namespace
}  // namespace attn

}  // namespace sph

using namespace sph;
using namespace sph::attn;

extern "C" int64_t sph_attention_scratch_bytes(const sph_attention* a, int backward) {
  Params p;
  const int rc = fill(a, __func__, &p);
  if (rc != SPH_OK) return rc;
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  const Plan plan = plan_of(*a, p, sms);
  const int64_t rows = (int64_t)p.n_q * p.hq, k_values = (int64_t)p.n_k * p.hkv * p.d;
  if (!backward) return plan.fwd.parts > 1 ? (plan.fwd.parts * rows * (p.d + 1) + rows) * 4 : 0;
  return 2 * (p.B + 2) * (int64_t)sizeof(ScanPlan) + ((rows + 3) / 4 * 4 + (std::max(rows, (int64_t)p.n_k * p.hkv) + 3) / 4 * 4 +
          std::max(plan.dq.parts > 1 ? plan.dq.parts * rows * p.d : 0, plan.dkv.parts > 1 ? 2 * plan.dkv.parts * k_values : 0)) * 4;
}

extern "C" int sph_attention_forward(const sph_attention* a, void* d_out, float* d_lse, void* d_scratch, int32_t* d_status, void* stream) {
  Params p;
  const int rc = fill(a, __func__, &p);
  if (rc != SPH_OK) return rc;
  if (a->n_q == 0) return SPH_OK;
  SPH_CHECK_ARG(d_out, "null pointer");
  SPH_CHECK_ARG(((uintptr_t)d_out & 15) == 0, "results must be 16-byte aligned");
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  const Plan plan = plan_of(*a, p, sms);
  SPH_CHECK_ARG(plan.fwd.parts == 1 || (d_scratch && (uintptr_t)d_scratch % 16 == 0), "the scratch must be 16-byte aligned");
  p.out = d_out;
  p.lse = d_lse;
  p.status = d_status;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool tc = on_tensor_cores(*a, p);
  if (a->dtype == SPH_F32) return run_forward<float>(p, plan, tc, d_scratch, st);
  if (a->dtype == SPH_F16) return run_forward<__half>(p, plan, tc, d_scratch, st);
  return run_forward<__nv_bfloat16>(p, plan, tc, d_scratch, st);
}

extern "C" int sph_attention_backward(const sph_attention* a, const void* d_dout, const void* d_out, const float* d_lse, void* d_scratch,
                                      void* d_dq, void* d_dk, void* d_dv, int32_t* d_status, void* stream) {
  Params p;
  const int rc = fill(a, __func__, &p);
  if (rc != SPH_OK) return rc;
  SPH_CHECK_ARG(a->n_q == 0 || (d_dout && d_out && d_lse), "null pointer");
  SPH_CHECK_ARG(!!d_dk == !!d_dv, "the gradients of keys and values come together");
  SPH_CHECK_ARG(d_scratch && (uintptr_t)d_scratch % 16 == 0, "the scratch must be 16-byte aligned");
  SPH_CHECK_ARG((((uintptr_t)d_dout | (uintptr_t)d_out | (uintptr_t)d_dq | (uintptr_t)d_dk | (uintptr_t)d_dv) & 15) == 0,
                "gradients and results must be 16-byte aligned");
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  const Plan plan = plan_of(*a, p, sms);
  p.d_out = d_dout;
  p.lse = const_cast<float*>(d_lse);
  p.dq = d_dq; p.dk = d_dk; p.dv = d_dv;
  p.status = d_status;
  const cudaStream_t st = (cudaStream_t)stream;
  const bool tc = on_tensor_cores(*a, p);
  if (a->dtype == SPH_F32) return run_backward<float>(p, plan, tc, d_out, d_scratch, st);
  if (a->dtype == SPH_F16) return run_backward<__half>(p, plan, tc, d_out, d_scratch, st);
  return run_backward<__nv_bfloat16>(p, plan, tc, d_out, d_scratch, st);
}
