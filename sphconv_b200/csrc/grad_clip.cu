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
constexpr int kBlocksPerSm = 8;

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
  int64_t begin, end;
  int src_dtype, dst_dtype;
};
__device__ __forceinline__ Piece piece_of(const Ranges& r, int chunk) {
  int lo = 0, hi = r.count - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (r.first[mid] <= chunk) lo = mid; else hi = mid - 1;
  }
  Piece p;
  p.src = r.src[lo];
  p.dst = r.dst[lo];
  p.begin = (int64_t)(chunk - r.first[lo]) * r.chunk;
  p.end = min(r.n[lo], p.begin + r.chunk);
  p.src_dtype = r.dtypes[lo] & 15;
  p.dst_dtype = r.dtypes[lo] >> 4;
  return p;
}

__device__ __forceinline__ float widen(unsigned short bits, int dtype) {
  return dtype == SPH_F16 ? __half2float(__ushort_as_half(bits)) : __uint_as_float((unsigned)bits << 16);
}
__device__ __forceinline__ unsigned short narrow(float v, int dtype) {
  return dtype == SPH_F16 ? __half_as_ushort(__float2half_rn(v)) : __bfloat16_as_ushort(__float2bfloat16_rn(v));
}

// Values i .. i+7 of a range (0 behind its end).  Plain loads: src may be dst.
__device__ __forceinline__ void load8(float (&v)[kVec], const void* src, int dtype, int64_t i, int64_t end) {
  const bool whole = i + kVec <= end;
  if (dtype == SPH_F32) {
    const float* s = (const float*)src + i;
    if (whole && ((uintptr_t)s & 15) == 0) {
      const float4 a = *(const float4*)s, b = *(const float4*)(s + 4);
      v[0] = a.x; v[1] = a.y; v[2] = a.z; v[3] = a.w; v[4] = b.x; v[5] = b.y; v[6] = b.z; v[7] = b.w;
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = i + j < end ? s[j] : 0.f;
    }
  } else {
    const unsigned short* s = (const unsigned short*)src + i;
    if (whole && ((uintptr_t)s & 15) == 0) {
      const uint4 a = *(const uint4*)s;
      const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        v[2 * j] = widen((unsigned short)(w[j] & 0xffffu), dtype);
        v[2 * j + 1] = widen((unsigned short)(w[j] >> 16), dtype);
      }
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] = i + j < end ? widen(s[j], dtype) : 0.f;
    }
  }
}

__device__ __forceinline__ void store8(const float (&v)[kVec], void* dst, int dtype, int64_t i, int64_t end) {
  const bool whole = i + kVec <= end;
  if (dtype == SPH_F32) {
    float* d = (float*)dst + i;
    if (whole && ((uintptr_t)d & 15) == 0) {
      *(float4*)d = make_float4(v[0], v[1], v[2], v[3]);
      *(float4*)(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < end) d[j] = v[j];
    }
  } else {
    unsigned short* d = (unsigned short*)dst + i;
    unsigned short h[kVec];
#pragma unroll
    for (int j = 0; j < kVec; ++j) h[j] = narrow(v[j], dtype);
    if (whole && ((uintptr_t)d & 15) == 0) {
      uint32_t w[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) w[j] = (uint32_t)h[2 * j] | (uint32_t)h[2 * j + 1] << 16;
      *(uint4*)d = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
      for (int j = 0; j < kVec; ++j)
        if (i + j < end) d[j] = h[j];
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
__global__ void __launch_bounds__(kThreads) norm_partials_kernel(const __grid_constant__ Ranges r, double* partial) {
  after_previous();
  double sum = 0.0;
  for (int c = blockIdx.x; c < r.chunks; c += gridDim.x) {
    const Piece p = piece_of(r, c);
    int64_t i = p.begin + (int64_t)threadIdx.x * kVec;
    for (; i < p.end; i += (int64_t)kThreads * kVec) {
      float v[kVec];
      load8(v, p.src, p.src_dtype, i, p.end);
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
    }
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
__global__ void __launch_bounds__(kThreads) clip_kernel(const __grid_constant__ Ranges r, const double* partial, int n, float max_norm,
                                                        float* norm) {
  after_previous();
  const float total = total_norm<MAX>(partial, n);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = total;
  float by = max_norm / (total + 1e-6f);
  if (by > 1.f) by = 1.f;                     // NaN stays
  for (int c = r.chunks - 1 - (int)blockIdx.x; c >= 0; c -= gridDim.x) {
    const Piece p = piece_of(r, c);
    if (by == 1.f && p.src == p.dst) continue;
    int64_t i = p.begin + (int64_t)threadIdx.x * kVec;
    for (; i < p.end; i += (int64_t)kThreads * kVec) {
      float v[kVec];
      load8(v, p.src, p.src_dtype, i, p.end);
#pragma unroll
      for (int j = 0; j < kVec; ++j) v[j] *= by;
      store8(v, p.dst, p.dst_dtype, i, p.end);
    }
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
  // chunks that give every block a few of them, so that none is left with much more than the others
  constexpr int64_t unit = kThreads * kVec;
  const int64_t per_block = total / ((int64_t)sms * kBlocksPerSm * 4);
  r->chunk = (int32_t)std::min<int64_t>(16 * unit, std::max<int64_t>(unit, div_up64(per_block, unit) * unit));
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
