// Global norm over many gradients, and clipping by it.
//
//   norm = sqrt(sum g^2) or max |g| over every value of every tensor;  dst = src * min(1, max_norm / (norm + 1e-6))
//
// Two launches for up to kBatch ranges of memory: partials (a number per block, summed in a fixed order: the same tensors give the same
// bits) and the scaling, every block of which adds the partials up again - a few KB from L2, cheaper than a third launch - and walks
// the ranges from their end, where what the first pass read last is still in L2.  Ranges that follow one another in memory are one
// range: a flat buffer's slices cost what the buffer costs.  Bound by HBM: every gradient is read twice (once from there where all of
// them fit L2) and written once.
//
// Sums of squares are held in 64 bits.  A group of 8 values is squared and summed in 32 bits first, at 2^-23 of the group's sum,
// unless that could over- or underflow: a conversion to 64 bits per value is 16 a cycle and SM, which is what HBM brings.
#include <algorithm>

#include "common.cuh"

namespace sph {

namespace {

constexpr int kThreads = 256;
constexpr int kVec = 8;                       // values a thread takes at a time: 16 bytes of a 16-bit type, 32 of float
constexpr int kBatch = 128;                   // ranges of a launch: their table is the kernel's argument (4 KB at most)
constexpr int kBlocksPerSm = 6;

struct Ranges {
  const void* src[kBatch];
  void* dst[kBatch];
  int64_t n[kBatch];
  int32_t first[kBatch];                      // its first chunk
  uint8_t dtypes[kBatch];                     // src | dst << 4
  int32_t count, chunks, chunk;               // chunk: values of one, a multiple of kThreads * kVec
};
static_assert(sizeof(Ranges) <= 4000, "kernel arguments are limited");

struct Piece {                                // one chunk of a range
  const void* src;
  void* dst;
  int n;
  int src_dtype, dst_dtype;
};
__device__ __forceinline__ int bytes_of(int dtype) { return dtype == SPH_F32 ? 4 : 2; }
__device__ __forceinline__ Piece piece_of(const Ranges& r, int chunk) {
  int lo = 0, hi = r.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (r.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  Piece p;
  const int64_t begin = (int64_t)(chunk - r.first[lo]) * r.chunk;
  p.src_dtype = r.dtypes[lo] & 15;
  p.dst_dtype = r.dtypes[lo] >> 4;
  p.src = (const char*)r.src[lo] + begin * bytes_of(p.src_dtype);
  p.dst = (char*)r.dst[lo] + begin * bytes_of(p.dst_dtype);
  p.n = (int)min(r.n[lo] - begin, (int64_t)r.chunk);
  return p;
}

__device__ __forceinline__ bool aligned(const void* p) { return ((uintptr_t)p & 15) == 0; }

// 8 values of a type, as they lie in memory.  Plain loads: src may be dst.
template <int DTYPE>
struct Eight {
  static constexpr int kWords = DTYPE == SPH_F32 ? 8 : 4;
  uint32_t w[kWords];
  __device__ __forceinline__ void fetch(const void* src, int i) {                // 16-byte aligned
    const uint4* s = (const uint4*)((const char*)src + (size_t)i * (DTYPE == SPH_F32 ? 4 : 2));
#pragma unroll
    for (int j = 0; j < kWords / 4; ++j) {
      const uint4 a = s[j];
      w[4 * j] = a.x; w[4 * j + 1] = a.y; w[4 * j + 2] = a.z; w[4 * j + 3] = a.w;
    }
  }
  __device__ __forceinline__ void fetch_some(const void* src, int i, int n) {    // any alignment, 0 from n on
    if (DTYPE == SPH_F32) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) w[j % kWords] = i + j < n ? ((const uint32_t*)src)[i + j] : 0u;
    } else {
      const unsigned short* s = (const unsigned short*)src + i;
#pragma unroll
      for (int j = 0; j < kVec / 2; ++j)
        w[j] = (i + 2 * j < n ? (uint32_t)s[2 * j] : 0u) | (i + 2 * j + 1 < n ? (uint32_t)s[2 * j + 1] << 16 : 0u);
    }
  }
  __device__ __forceinline__ void values(float (&v)[kVec]) const {
#pragma unroll
    for (int j = 0; j < kVec; ++j) {
      if (DTYPE == SPH_F32) {
        v[j] = __uint_as_float(w[j % kWords]);
      } else if (DTYPE == SPH_BF16) {
        v[j] = __uint_as_float(j & 1 ? w[j / 2] & 0xffff0000u : w[j / 2] << 16);
      } else {
        const float2 f = __half22float2(*(const __half2*)&w[j / 2]);
        v[j] = j & 1 ? f.y : f.x;
      }
    }
  }
};

// f(values, place of the first) for every 8 values of a piece that are this thread's, kAhead times as many asked for at once.
constexpr int kAhead = 4;
template <int DTYPE, typename F>
__device__ __forceinline__ void each(const Piece& p, F f) {
  constexpr int step = kThreads * kVec;
  int i = (int)threadIdx.x * kVec;
  float v[kVec];
  if (aligned(p.src)) {
    const int last = p.n - kVec;              // the last place of 8 values
    for (; i + (kAhead - 1) * step <= last; i += kAhead * step) {
      Eight<DTYPE> r[kAhead];
#pragma unroll
      for (int a = 0; a < kAhead; ++a) r[a].fetch(p.src, i + a * step);
#pragma unroll
      for (int a = 0; a < kAhead; ++a) {
        r[a].values(v);
        f(v, i + a * step);
      }
    }
#pragma unroll 1
    for (; i <= last; i += step) {
      Eight<DTYPE> r;
      r.fetch(p.src, i);
      r.values(v);
      f(v, i);
    }
  }
#pragma unroll 1
  for (; i < p.n; i += step) {
    Eight<DTYPE> r;
    r.fetch_some(p.src, i, p.n);
    r.values(v);
    f(v, i);
  }
}
template <typename F>
__device__ __forceinline__ void each(const Piece& p, F f) {
  if (p.src_dtype == SPH_F32) each<SPH_F32>(p, f);
  else if (p.src_dtype == SPH_F16) each<SPH_F16>(p, f);
  else each<SPH_BF16>(p, f);
}

__device__ __forceinline__ uint32_t narrow(float a, float b, int dtype) {
  if (dtype == SPH_F16) {
    const __half2 h = __floats2half2_rn(a, b);
    return *(const uint32_t*)&h;
  }
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *(const uint32_t*)&h;
}
// Values i .. i+7 of a piece, those that there are.
__device__ __forceinline__ void store8(const float (&v)[kVec], const Piece& p, int i, bool dst_aligned) {
  if (p.dst_dtype == SPH_F32) {
    float* d = (float*)p.dst + i;
    if (dst_aligned && i + kVec <= p.n) {
      *(float4*)d = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < p.n) d[j] = v[j];
    }
  } else {
    unsigned short* d = (unsigned short*)p.dst + i;
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) w[j] = narrow(v[2 * j], v[2 * j + 1], p.dst_dtype);
    if (dst_aligned && i + kVec <= p.n) {
      *(uint4*)d = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < p.n) d[j] = (unsigned short)(w[j / 2] >> (16 * (j & 1)));
    }
  }
}

// Sum (MAX: largest, NaN above all) over a block, in an order that depends on the thread numbers alone; in every thread.
template <bool MAX>
__device__ __forceinline__ double join(double a, double b) {
  if (!MAX) return a + b;
  return (a >= b || a != a) ? a : b;
}
template <bool MAX>
__device__ double block_join(double v) {
  __shared__ double s[kThreads / 32];
  for (int o = 16; o > 0; o >>= 1) v = join<MAX>(v, __shfl_xor_sync(0xffffffffu, v, o));
  if ((threadIdx.x & 31) == 0) s[threadIdx.x >> 5] = v;
  __syncthreads();
  v = s[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) v = join<MAX>(v, s[w]);
  return v;
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) norm_partials_kernel(const __grid_constant__ Ranges r, double* partial) {
  after_previous();
  double sum = 0.0;
  for (int c = blockIdx.x; c < r.chunks; c += gridDim.x) {
    const Piece p = piece_of(r, c);
    each(p, [&](float (&v)[kVec], int) {
      if (MAX) {
        unsigned top = 0u;                    // as integers |NaN| is above infinity
#pragma unroll
        for (int j = 0; j < kVec; ++j) top = max(top, __float_as_uint(v[j]) & 0x7fffffffu);
        sum = join<true>(sum, (double)__uint_as_float(top));
      } else {
        float t = 0.f;
#pragma unroll
        for (int j = 0; j < kVec; ++j) t = fmaf(v[j], v[j], t);
        if (t > 1e-24f && t < 1e37f) {        // squares below 1e-38 that were lost are below 2^-43 of it
          sum += (double)t;
        } else {
#pragma unroll
          for (int j = 0; j < kVec; ++j) sum = fma((double)v[j], (double)v[j], sum);
        }
      }
    });
  }
  sum = block_join<MAX>(sum);
  if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

template <bool MAX>
__device__ float total_norm(const double* partial, int n) {
  double sum = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) sum = join<MAX>(sum, partial[i]);
  sum = block_join<MAX>(sum);
  return (float)(MAX ? sum : sqrt(sum));
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads) norm_kernel(const double* partial, int n, float* norm) {
  after_previous();
  const float total = total_norm<MAX>(partial, n);
  if (threadIdx.x == 0) *norm = total;
}

template <bool MAX>
__global__ void __launch_bounds__(kThreads, kBlocksPerSm) clip_kernel(const __grid_constant__ Ranges r, const double* partial, int n, float max_norm,
                                                        float* norm) {
  after_previous();
  const float total = total_norm<MAX>(partial, n);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  float by = max_norm / (total + 1e-6f);
  if (by > 1.f) by = 1.f;                     // NaN stays
  for (int c = r.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const Piece p = piece_of(r, c);
    if (by == 1.f && p.src == p.dst) continue;
    const bool dst_aligned = aligned(p.dst);
    each(p, [&](float (&v)[kVec], int i) {
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] *= by;
      store8(v, p, i, dst_aligned);
    });
  }
}

int esize_of(int dtype) { return dtype == SPH_F32 ? 4 : dtype == SPH_F16 || dtype == SPH_BF16 ? 2 : 0; }

// The next ranges from tensor *at on, those that follow one another in memory as one.  with_dst: the destinations have to as well.
int64_t take(const sph_clip_tensor* t, int32_t count, int32_t* at, bool with_dst, int sms, Ranges* r, unsigned* grid) {
  r->count = 0;
  int64_t total = 0;
  for (; *at < count; ++*at) {
    const sph_clip_tensor& x = t[*at];
    if (x.n == 0) continue;
    const uint8_t types = (uint8_t)(x.src_dtype | (with_dst ? x.dst_dtype : 0) << 4);
    const int k = r->count - 1;
    const bool follows = k >= 0 && r->dtypes[k] == types &&
                         (const char*)r->src[k] + r->n[k] * esize_of(x.src_dtype) == (const char*)x.src &&
                         (!with_dst || (char*)r->dst[k] + r->n[k] * esize_of(x.dst_dtype) == (char*)x.dst);
    if (follows) {
      r->n[k] += x.n;
    } else {
      if (r->count == kBatch) break;
      r->src[r->count] = x.src;
      r->dst[r->count] = with_dst ? x.dst : nullptr;
      r->n[r->count] = x.n;
      r->dtypes[r->count++] = types;
    }
    total += x.n;
  }
  // chunks that give every block some of them, so that none is left with much more than the others
  constexpr int64_t unit = kThreads * kVec;
  const int64_t per_block = total / ((int64_t)sms * kBlocksPerSm * 6);
  const int64_t whole = per_block >= kAhead * unit ? kAhead * unit : unit;
  r->chunk = (int32_t)std::min<int64_t>(64 * unit, std::max<int64_t>(unit, div_up64(per_block, whole) * whole));
  int64_t chunks = 0;
  for (int k = 0; k < r->count; ++k) {
    r->first[k] = (int32_t)chunks;
    chunks += div_up64(r->n[k], r->chunk);
    if (chunks > INT32_MAX) return -1;
  }
  r->chunks = (int32_t)chunks;
  *grid = (unsigned)std::min<int64_t>(chunks, (int64_t)sms * kBlocksPerSm);
  return total;
}

int grad_clip(const sph_clip_tensor* tensors, int32_t count, int norm_kind, bool clip, float max_norm, void* scratch, float* d_norm,
        cudaStream_t st) {
  SPH_CHECK_ARG(count >= 0 && (count == 0 || tensors), "bad list of tensors");
  SPH_CHECK_ARG(d_norm, "null pointer");
  SPH_CHECK_ARG(norm_kind == SPH_NORM_2 || norm_kind == SPH_NORM_MAX, "the norm is SPH_NORM_2 or SPH_NORM_MAX");
  SPH_CHECK_ARG(!clip || max_norm >= 0.f, "max_norm must not be negative or NaN");
  for (int32_t i = 0; i < count; ++i) {
    const sph_clip_tensor& t = tensors[i];
    SPH_CHECK_ARG(t.n >= 0 && (t.n == 0 || (t.src && (!clip || t.dst))), "bad tensor");
    SPH_CHECK_ARG(esize_of(t.src_dtype) && (!clip || esize_of(t.dst_dtype)), "gradients are fp32, fp16 or bf16");
    SPH_CHECK_ARG((uintptr_t)t.src % esize_of(t.src_dtype) == 0 && (!clip || (uintptr_t)t.dst % esize_of(t.dst_dtype) == 0),
                  "a tensor is not aligned to its elements");
  }
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  SPH_CHECK_ARG(scratch && (uintptr_t)scratch % 8 == 0, "the scratch must be 8-byte aligned");
  double* partial = (double*)scratch;
  int n = 0;
  const bool max = norm_kind == SPH_NORM_MAX;
  Ranges r;
  unsigned grid;
  for (int32_t at = 0; at < count;) {
    const int64_t total = take(tensors, count, &at, false, sms, &r, &grid);
    if (total < 0) { set_error("%s: too many values", __func__); return SPH_ERR_LIMIT; }
    if (total == 0) continue;
    if (max) launch(norm_partials_kernel<true>, grid, kThreads, 0, st, r, partial + n);
    else launch(norm_partials_kernel<false>, grid, kThreads, 0, st, r, partial + n);
    SPH_LAUNCH_CHECK();
    n += (int)grid;
  }
  bool written = false;
  if (clip) {
    for (int32_t at = 0; at < count;) {
      const int64_t total = take(tensors, count, &at, true, sms, &r, &grid);
      if (total < 0) { set_error("%s: too many values", __func__); return SPH_ERR_LIMIT; }
      if (total == 0) continue;
      if (max) launch(clip_kernel<true>, grid, kThreads, 0, st, r, partial, n, max_norm, d_norm);
      else launch(clip_kernel<false>, grid, kThreads, 0, st, r, partial, n, max_norm, d_norm);
      SPH_LAUNCH_CHECK();
      written = true;
    }
  }
  if (!written) {
    if (max) launch(norm_kernel<true>, 1, kThreads, 0, st, partial, n, d_norm);
    else launch(norm_kernel<false>, 1, kThreads, 0, st, partial, n, d_norm);
    SPH_LAUNCH_CHECK();
  }
  return SPH_OK;
}

}  // namespace

}  // namespace sph

using namespace sph;

extern "C" int64_t sph_grad_norm_scratch_bytes(int32_t count) {
  if (count < 0) { set_error("%s: bad count", __func__); return SPH_ERR_INVALID; }
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  return (int64_t)div_up(count > 0 ? count : 1, kBatch) * sms * kBlocksPerSm * (int64_t)sizeof(double);
}

extern "C" int sph_grad_norm(const sph_clip_tensor* tensors, int32_t count, int norm_kind, void* d_scratch, float* d_norm, void* stream) {
  return grad_clip(tensors, count, norm_kind, false, 0.f, d_scratch, d_norm, (cudaStream_t)stream);
}

extern "C" int sph_grad_clip(const sph_clip_tensor* tensors, int32_t count, int norm_kind, float max_norm, void* d_scratch, float* d_norm,
                             void* stream) {
  return grad_clip(tensors, count, norm_kind, true, max_norm, d_scratch, d_norm, (cudaStream_t)stream);
}
