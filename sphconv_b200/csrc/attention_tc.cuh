// What the tensor-core kernels of the cross attention share: operand tiles in shared memory and their descriptors, TMEM helpers, loads.
//
// A tile is `rows` rows of up to 64 or 128 channels, in blocks of 64 channels: a block is rows x 128 bytes with the 128-byte
// swizzle (16-byte piece c of row r at 128 r + 16 (c ^ (r & 7))).  The same tile is an operand along its channels (K-major: scores) and
// along its rows (MN-major: products with P or dS).
#pragma once

#include <cuda.h>

#include <type_traits>

#include "attention.cuh"
#include "tc_common.cuh"

namespace sph {
namespace attn {

using namespace tc;

constexpr int kM = 128;                       // rows of a tile: the lanes of TMEM

// Descriptor of a tile at `addr` (1024-byte aligned).  K-major: 8 rows lie 1024 bytes apart, the next 16 channels of a
// block 32 bytes on.  MN-major: `lbo` bytes between blocks of 64 channels, 1024 between 8 rows; 16 rows are 2048 bytes.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, uint32_t lbo) {
  return make_smem_desc(addr, lbo, 1024u) | (uint64_t)2 << 61;
}

// A in TMEM (16-bit elements, two to a column), B in shared memory.
__device__ __forceinline__ void umma_f16_ta(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem), "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate));
}

// 32 consecutive columns of this thread's TMEM lane.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]),
        "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]),
        "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]),
        "=r"(v[30]), "=r"(v[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]),
      "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]),
      "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,"
      "%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]),
      "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
      "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
      "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st8(uint32_t taddr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]),
               "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float max3(float a, float b, float c) {
  float y;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(y) : "f"(a), "f"(b), "f"(c));
  return y;
}

// Two values rounded to the rows' type, the first in the lower half.
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  if (BF16) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *(const uint32_t*)&v;
  }
  const __half2 v = __floats2half2_rn(a, b);
  return *(const uint32_t*)&v;
}
template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t w) {
  if (BF16) return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
  return __half22float2(*(const __half2*)&w);
}

// Rows of one head, or of the heads of a group, as TMA brings them to a tile: blocks of 64 channels, zeros behind the last one.
struct TileMap {
  CUtensorMap map;                            // [heads][rows] or [rows][heads] of channels, the smaller stride inside
  int rows_inside;
  int usable;                                 // 0: strides or a group that a map cannot have; rows are copied with cp.async
};

// Rows `first` on of `head` to the tile at `to`, whose blocks are `block` bytes; by one thread, which has announced the bytes.
template <int DP>
__device__ __forceinline__ void tma_tile(uint32_t to, uint32_t block, const TileMap& m, int head, int first, uint32_t bar) {
  const int a = m.rows_inside ? first : head, b = m.rows_inside ? head : first;
#pragma unroll
  for (int x = 0; x < DP; x += 64)
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
            to + (uint32_t)(x / 64) * block),
        "l"(&m.map), "r"(x), "r"(a), "r"(b), "r"(bar)
        : "memory");
}

// The barrier gets an arrival more, which comes when this thread's copies so far have landed: the warp's own arrival follows at once.
__device__ __forceinline__ void cp_async_arrive(uint32_t bar) {
  asm volatile("cp.async.mbarrier.arrive.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}

// How `threads` loading threads share a tile's 16-byte pieces: `lanes` of them (a power of two) a row.
struct Pieces {
  int pieces;                                 // of a row: channels in steps of 16, two pieces each
  int shift;                                  // lanes = 1 << shift
};
__device__ __forceinline__ Pieces pieces_of(int d) {
  Pieces r;
  r.pieces = (d + 15) / 16 * 2;
  r.shift = r.pieces <= 2 ? 1 : r.pieces <= 4 ? 2 : r.pieces <= 8 ? 3 : 4;
  return r;
}

// Rows 0 .. n-1 of a tile of ROWS rows by THREADS threads with cp.async, zeros from n on, behind d channels, and where ok(r) is false;
// row(r) is the address of row r's channels.
template <int ROWS, int THREADS, typename Row, typename Ok>
__device__ __forceinline__ void load_rows(uint32_t to, int t, int n, int d, const Pieces& pc, const void* any, Row row, Ok ok) {
  const int c = t & ((1 << pc.shift) - 1), step = THREADS >> pc.shift;
  if (c >= pc.pieces) return;
  const uint32_t block = to + (uint32_t)(c >> 3) * (ROWS * 128u);
  const bool inside = c * 8 < d;
#pragma unroll 4
  for (int r = t >> pc.shift; r < ROWS; r += step) {
    const bool some = inside && r < n && ok(r);
    const uint32_t dst = block + (uint32_t)r * 128u + (uint32_t)(((c & 7) ^ (r & 7)) << 4);
    cp_async_16(dst, some ? (const uint8_t*)row(r) + c * 16 : (const uint8_t*)any, some ? 16u : 0u);
  }
}

// 16 accumulator values times `by` to 16-bit or float32 memory that is 16-byte aligned in steps of 8 (16-bit) or 4 values; all 16 of a
// 16-bit type in one store where the address is a multiple of 32.
template <bool BF16>
__device__ __forceinline__ void store16(const uint32_t (&v)[16], float by, void* to, int n) {       // n: of them, a multiple of 8
  uint32_t w[8];
#pragma unroll
  for (int j = 0; j < 8; ++j) w[j] = pack2<BF16>(__uint_as_float(v[2 * j]) * by, __uint_as_float(v[2 * j + 1]) * by);
  if (n >= 16 && ((uintptr_t)to & 31) == 0) {
    asm volatile("st.global.v8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"l"(to), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]),
                 "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
    return;
  }
  ((uint4*)to)[0] = make_uint4(w[0], w[1], w[2], w[3]);
  if (n >= 16) ((uint4*)to)[1] = make_uint4(w[4], w[5], w[6], w[7]);
}
__device__ __forceinline__ void store16_float(const uint32_t (&v)[16], float by, float* to, int n) {
  float4* dst = (float4*)to;
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    if (4 * i >= n) break;
    dst[i] = make_float4(__uint_as_float(v[4 * i]) * by, __uint_as_float(v[4 * i + 1]) * by, __uint_as_float(v[4 * i + 2]) * by,
                         __uint_as_float(v[4 * i + 3]) * by);
  }
}

// Which of the 64 keys from `first` on, of `n`, are some: bit i of word w is key 32 w + i.  By whole warps.
__device__ __forceinline__ uint2 key_bits(const uint8_t* mask, int64_t first, int n) {
  const int lane = threadIdx.x & 31;
  uint32_t w[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int r = 32 * i + lane;
    w[i] = __ballot_sync(0xffffffffu, r < n && (mask == nullptr || __ldg(mask + first + r) != 0));
  }
  return make_uint2(w[0], w[1]);
}

// Host: a map of x [rows][heads][d] with strides in elements, for tiles of `tile` rows of a head, or (group > 1) of the rows of `group`
// heads taken together.
void make_tile_map(TileMap* m, const void* x, int64_t rows, int heads, int d, int64_t row_stride, int64_t head_stride, int tile, int group);

// What a kernel does when a wait ran out, in front of its last barrier: report, and let what is in flight end.
__device__ __forceinline__ void wind_down(volatile int* aborted, int* status) {
  if (!*aborted) return;
  cp_async_wait_all();
  const long long t0 = clock64();
  while (clock64() - t0 < 4000000ll) { }
  if (threadIdx.x == 0 && status) atomicOr(status, SPH_STATUS_TIMEOUT);
}

}  // namespace attn
}  // namespace sph
