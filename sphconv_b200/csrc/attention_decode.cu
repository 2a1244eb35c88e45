// Cross attention of a few queries a scan, the decoding step: keys and values are read once and everything else is small, so the bound is
// HBM.  A block has up to R query rows of one key head and a part of the keys.  LANES lanes have a key, 16 bytes of it each, and all R
// rows' slices of those channels; a warp takes 2 * 32 / LANES keys at a time, and has three times as many on their way to shared memory, where
// every lane finds its own: asked for into registers, four keys a lane left HBM at 47 %.  Every group of lanes has
// its own softmax - maximum, sum and O - over the keys it saw; they are joined at the end, over the warp, the block and, where the keys are
// split over blocks, in a second launch.  The maximum follows only when a score is more than 2^8 above it.
//
// Exponentials are approximate, to 2^-22 of P, in float32 as well: four steps of float32, and less than what rounding leaves in a score of
// 4 or more (the results of 700 float32 rows are off by 2.3e-7 of their size, where float32 operations one by one leave 1.8e-7).  P itself
// is never rounded to 16 bits here.
//
// The sum over a key's lanes leaves each lane the scores of its share of the rows, whose powers it takes alone and hands round.
// One query over 87 k rows of 8 scans, 8 key heads of 64 channels, bf16: 235 us, 6.1 TB/s.  With 4 rows a key head the instructions take
// longer than the loads (2 key heads: 95 us, on the tensor cores, whose tiles of 128 rows then have 4, 84; 128 channels 170 and 139),
// so 16-bit keys come here for one row only; float32, whose other kernel has tiles of 64 rows on the CUDA cores, for up to 8.
// Lengths are on the device only, so this goes by the rows of a scan on average: where one of many scans has them all, its keys are read
// once a row (64 queries over 87 k rows, 8 heads of 64, bf16: 1636 us beside 63 scans without queries, 48 alone).
#include <algorithm>

#include "attention.cuh"
#include "tc_common.cuh"

namespace sph {
namespace attn {

namespace {

constexpr int kWarps = 8, kThreadsDecode = kWarps * 32;
constexpr int kKeys = 2, kStages = 4;         // keys of a lane a stage, and stages
constexpr int kStep = 64;                     // parts are whole steps of so many keys
constexpr float kSlack = 8.f;

template <typename T> struct Key;             // 16 bytes of a row as pairs
template <> struct Key<float> {
  static constexpr int kPairs = 2;
  static __device__ __forceinline__ void pairs(float2 (&x)[2], const uint4& w) {
    x[0] = make_float2(__uint_as_float(w.x), __uint_as_float(w.y));
    x[1] = make_float2(__uint_as_float(w.z), __uint_as_float(w.w));
  }
  static __device__ __forceinline__ float put(float v) { return v; }
};
template <> struct Key<__half> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ void pairs(float2 (&x)[4], const uint4& w) {
    x[0] = __half22float2(*(const __half2*)&w.x);
    x[1] = __half22float2(*(const __half2*)&w.y);
    x[2] = __half22float2(*(const __half2*)&w.z);
    x[3] = __half22float2(*(const __half2*)&w.w);
  }
  static __device__ __forceinline__ __half put(float v) { return __float2half_rn(v); }
};
template <> struct Key<__nv_bfloat16> {
  static constexpr int kPairs = 4;
  static __device__ __forceinline__ float2 two(uint32_t w) { return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u)); }
  static __device__ __forceinline__ void pairs(float2 (&x)[4], const uint4& w) {
    x[0] = two(w.x); x[1] = two(w.y); x[2] = two(w.z); x[3] = two(w.w);
  }
  static __device__ __forceinline__ __nv_bfloat16 put(float v) { return __float2bfloat16_rn(v); }
};

__device__ __forceinline__ float2 twice(float v) { return make_float2(v, v); }

// The softmax of two sets of keys as one: a row's maximum, sum and part of O.
template <int P>
__device__ __forceinline__ void join(float& m, float& l, float2 (&o)[P], float m2, float l2, const float2 (&o2)[P]) {
  const float top = fmaxf(m, m2), base = top == -INFINITY ? 0.f : top;
  const float a = exp2f(m - base), b = exp2f(m2 - base);
#pragma unroll
  for (int i = 0; i < P; ++i) o[i] = fma2(o2[i], twice(b), mul2(o[i], twice(a)));
  l = l * a + l2 * b;
  m = top;
}

template <typename T, int LANES, int R>
__global__ void __launch_bounds__(kThreadsDecode, 2) decode_kernel(const __grid_constant__ Params p) {
  constexpr int P = Key<T>::kPairs, E = 2 * P, KEYS = 32 / LANES;
  __shared__ Work s_work;
  __shared__ float s_m[kWarps][R], s_l[kWarps][R];
  __shared__ __align__(16) float s_o[kWarps][R][LANES * E];           // written two at a time
  after_previous();
  report_scans(p);
  const int head = blockIdx.x % p.hkv;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  if (warp == 0) {
    const Work w = find_work<true>(p, blockIdx.x / p.hkv, R, kStep);
    if (lane == 0) s_work = w;
  }
  __syncthreads();
  const Work w = s_work;
  if (w.scan < 0) return;
  const int rows = min(R, w.nq * p.group - w.tile * R);
  const int c = lane % LANES;                 // this lane's 16 bytes of a row
  const bool inside = c * E < p.d;
  auto out_row = [&](int r) {                 // of [n_q][hq]
    const int i = w.tile * R + r;
    return (int64_t)(w.q0 + i / p.group) * p.hq + head * p.group + i % p.group;
  };
  constexpr int W = R > LANES ? R / LANES : 1;             // rows whose softmax a lane has: W * ((c * R) / (LANES * W)) on
  float2 q[R][P], o[R][P];
  float m[W], l[W];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    uint4 x = make_uint4(0u, 0u, 0u, 0u);
    if (r < rows && inside) {
      const int i = w.tile * R + r;
      x = __ldg((const uint4*)((const T*)p.q + (int64_t)(w.q0 + i / p.group) * p.q_row + (head * p.group + i % p.group) * p.q_head) + c);
    }
    Key<T>::pairs(q[r], x);
#pragma unroll
    for (int i = 0; i < P; ++i) {
      q[r][i] = mul2(q[r][i], twice(p.scale_log2));
      o[r][i] = twice(0.f);
    }
  }
#pragma unroll
  for (int i = 0; i < W; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }
  // of value i % W of every lane that has row r
  auto of_row = [&](const float (&x)[W], int r) { return __shfl_sync(0xffffffffu, x[r % W], r / W * (LANES * W / R), LANES); };
  const int2 keys = make_int2(w.first, w.last);
  const T* k_at = (const T*)p.k + (int64_t)w.k0 * p.k_row + head * p.k_head;
  const T* v_at = (const T*)p.v + (int64_t)w.k0 * p.v_row + head * p.v_head;
  const int mine = warp * KEYS + lane / LANES;
  constexpr int step = kWarps * KEYS;
  extern __shared__ __align__(16) uint4 s_keys[];           // [warps][stages][keys][K, V][32]
  uint4* own = s_keys + warp * (kStages * kKeys * 2 * 32) + lane;
  auto is_key = [&](int k) { return k < keys.y && (p.mask == nullptr || __ldg(p.mask + (int64_t)w.k0 + k) != 0); };
  auto ask = [&](int stage, int base) {                     // what is no key is zeros: its values may be anything
#pragma unroll
    for (int a = 0; a < kKeys; ++a) {
      const int k = base + a * step + mine;
      const bool some = inside && is_key(k);
      const uint32_t to = tc::smem_u32(own + (stage * kKeys + a) * 64), bytes = some ? 16u : 0u;
      tc::cp_async_16(to, some ? (const uint4*)(k_at + (int64_t)k * p.k_row) + c : (const uint4*)p.k, bytes);
      tc::cp_async_16(to + 512u, some ? (const uint4*)(v_at + (int64_t)k * p.v_row) + c : (const uint4*)p.v, bytes);
    }
  };
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) {
    if (keys.x + i * kKeys * step < keys.y) ask(i, keys.x + i * kKeys * step);
    tc::cp_async_commit();
  }
  int stage = 0;
  for (int base = keys.x; base < keys.y; base += kKeys * step, stage = (stage + 1) % kStages) {
    const int later = base + (kStages - 1) * kKeys * step;
    if (later < keys.y) ask((stage + kStages - 1) % kStages, later);
    tc::cp_async_commit();
    asm volatile("cp.async.wait_group %0;" ::"n"(kStages - 1) : "memory");        // a lane reads what it asked for itself
#pragma unroll
    for (int a = 0; a < kKeys; ++a) {
      const bool key = is_key(base + a * step + mine);
      float2 x[P], v[P];
      Key<T>::pairs(x, own[(stage * kKeys + a) * 64]);
      Key<T>::pairs(v, own[(stage * kKeys + a) * 64 + 32]);
      float s[R];
#pragma unroll
      for (int r = 0; r < R; ++r) {
        float2 t = mul2(q[r][0], x[0]);
#pragma unroll
        for (int i = 1; i < P; ++i) t = fma2(q[r][i], x[i], t);
        s[r] = t.x + t.y;
      }
      // sums over the key's lanes: every step halves the rows that a lane goes on with
      int have = R;
#pragma unroll
      for (int of = LANES / 2; of > 0; of >>= 1) {
        if (have > 1) {
          const int half = have / 2;
          const bool upper = (lane & of) != 0;
#pragma unroll
          for (int i = 0; i < R / 2; ++i)
            if (i < half) {
              const float give = upper ? s[i] : s[i + half], keep = upper ? s[i + half] : s[i];
              s[i] = keep + __shfl_xor_sync(0xffffffffu, give, of);
            }
          have = half;
        } else {
          s[0] += __shfl_xor_sync(0xffffffffu, s[0], of);
        }
      }
      bool above = false;
#pragma unroll
      for (int i = 0; i < W; ++i) {
        s[i] = key ? s[i] : -INFINITY;
        above |= s[i] > m[i] + kSlack;
      }
      if (__any_sync(0xffffffffu, above)) {
        float by[W];
#pragma unroll
        for (int i = 0; i < W; ++i) {
          by[i] = 1.f;
          if (s[i] > m[i] + kSlack) {
            by[i] = exp2_approx(m[i] - s[i]);
            l[i] *= by[i];
            m[i] = s[i];
          }
        }
#pragma unroll
        for (int r = 0; r < R; ++r) {
          const float f = of_row(by, r);
#pragma unroll
          for (int i = 0; i < P; ++i) o[r][i] = mul2(o[r][i], twice(f));
        }
      }
      float e[W];
#pragma unroll
      for (int i = 0; i < W; ++i) {
        e[i] = exp2_approx(s[i] - (m[i] == -INFINITY ? 0.f : m[i]));
        l[i] += e[i];
      }
#pragma unroll
      for (int r = 0; r < R; ++r) {
        const float f = of_row(e, r);
#pragma unroll
        for (int i = 0; i < P; ++i) o[r][i] = fma2(twice(f), v[i], o[r][i]);
      }
    }
  }
  float row_m[R], row_l[R];
#pragma unroll
  for (int r = 0; r < R; ++r) {
    row_m[r] = of_row(m, r);
    row_l[r] = of_row(l, r);
  }
#pragma unroll
  for (int of = LANES; of < 32; of <<= 1)
#pragma unroll
    for (int r = 0; r < R; ++r) {
      float2 o2[P];
#pragma unroll
      for (int i = 0; i < P; ++i)
        o2[i] = make_float2(__shfl_xor_sync(0xffffffffu, o[r][i].x, of), __shfl_xor_sync(0xffffffffu, o[r][i].y, of));
      const float m2 = __shfl_xor_sync(0xffffffffu, row_m[r], of), l2 = __shfl_xor_sync(0xffffffffu, row_l[r], of);
      join(row_m[r], row_l[r], o[r], m2, l2, o2);
    }
  if (lane < LANES) {
#pragma unroll
    for (int r = 0; r < R; ++r) {
      if (lane == 0) {
        s_m[warp][r] = row_m[r];
        s_l[warp][r] = row_l[r];
      }
#pragma unroll
      for (int i = 0; i < P; ++i) *(float2*)&s_o[warp][r][c * E + 2 * i] = o[r][i];
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < rows * LANES * E; i += kThreadsDecode) {
    const int r = i / (LANES * E), ch = i % (LANES * E);
    float top = -INFINITY, sum = 0.f, v = 0.f;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) top = fmaxf(top, s_m[x][r]);
    const float base = top == -INFINITY ? 0.f : top;
#pragma unroll
    for (int x = 0; x < kWarps; ++x) {
      const float f = exp2f(s_m[x][r] - base);
      sum += f * s_l[x][r];
      v = fmaf(f, s_o[x][r][ch], v);
    }
    const bool none = sum == 0.f;
    const int64_t at = out_row(r), part_at = (int64_t)w.part * p.n_q * p.hq + at;
    if (ch < p.d) {
      const float result = none ? 0.f : v / sum;
      if (p.parts > 1) p.part[part_at * p.d + ch] = result;
      else ((T*)p.out)[at * p.d + ch] = Key<T>::put(result);
    }
    if (ch == 0) {
      const float lse = none ? INFINITY : top + log2f(sum);
      if (p.parts > 1 && w.part == 0) p.part_count[at] = w.parts;
      if (p.parts > 1) p.part_lse[part_at] = lse;
      else if (p.lse) p.lse[at] = lse;
    }
  }
}

template <typename T, int LANES, int R>
int start(const Params& p, int blocks, cudaStream_t st) {
  constexpr int smem = kWarps * kStages * kKeys * 2 * 32 * 16;
  SPH_CUDA(allow_smem(decode_kernel<T, LANES, R>, smem));
  launch(decode_kernel<T, LANES, R>, blocks, kThreadsDecode, smem, st, p);
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}
template <typename T, int R>
int start(const Params& p, int blocks, cudaStream_t st) {
  const int lanes = div_up(p.d * (int)sizeof(T), 16);
  if (lanes <= 4) return start<T, 4, R>(p, blocks, st);
  if (lanes <= 8) return start<T, 8, R>(p, blocks, st);
  if (lanes <= 16) return start<T, 16, R>(p, blocks, st);
  if constexpr (sizeof(T) == 4) return start<T, 32, R>(p, blocks, st);
  set_error("attention_decode: unsupported number of channels");
  return SPH_ERR_UNSUPPORTED;
}

}  // namespace

// Most query rows of a block, for `rows` of a scan and key head on average; 0: too many for this kernel.
int attention_decode_rows(int dtype, int64_t rows) { return rows <= 1 ? 1 : dtype == SPH_F32 && rows <= 8 ? 8 : 0; }

int attention_decode(const Params& p, int dtype, int rows, int blocks, cudaStream_t st) {
  if (dtype == SPH_F32) return rows == 1 ? start<float, 1>(p, blocks, st) : start<float, 8>(p, blocks, st);
  return dtype == SPH_F16 ? start<__half, 1>(p, blocks, st) : start<__nv_bfloat16, 1>(p, blocks, st);
}

}  // namespace attn
}  // namespace sph
