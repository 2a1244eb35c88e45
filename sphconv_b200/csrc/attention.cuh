// What the kernels of the cross attention share: their parameters, and how a block finds its work.
//
// Queries and keys are rows of B scans; scan b has the rows ptr[b] .. ptr[b+1]-1 of each, and what lies in front of the first or behind
// the last scan is treated as two scans more that have nothing on the other side: such rows get zeros.  The lengths are on the device
// only.  A grid has room for as many tiles as any lengths could need, and every block counts through the scans to find its own.
//
// Query heads that share a key head are rows of one tile: row r of a scan and key head is query r / group, head r % group.
#pragma once

#include "common.cuh"

namespace sph {
namespace attn {

constexpr float kLog2e = 1.4426950408889634f;

struct Params {
  const void *q, *k, *v;
  int64_t q_row, q_head, k_row, k_head, v_row, v_head;      // strides, in elements
  const int *q_ptr, *k_ptr;                                 // [B+1]
  const uint8_t* mask;                                      // [n_k], zero: no key; or null
  int n_q, n_k, B, hq, hkv, group, d;
  float scale, scale_log2;
  void* out;                                                // [n_q][hq][d]
  float* lse;                                               // [n_q][hq] log2 of a row's sum of 2^score, +inf: no keys
  const void* d_out;                                        // [n_q][hq][d]
  const float* delta;                                       // [n_q][hq] sum of d_out * out
  void *dq, *dk, *dv;                                       // as q, [n_k][hkv][d]
  float *part, *part2;                                      // with splits > 1: [splits][rows][heads][d], and of dv
  float* part_lse;                                          // forward: [splits][n_q][hq]
  int splits;
  int vec;                                                  // rows can be read in pieces of 16 bytes
  int* status;
};

// One tile of queries or keys.
struct Work {
  int scan;                                                 // -1: nothing to do
  int tile;
  int q0, nq, k0, nk;                                       // rows of the scan
};

__device__ __forceinline__ int2 scan_rows(const int* ptr, int B, int n, int s) {
  const int begin = s == 0 ? 0 : min(max(__ldg(ptr + s - 1), 0), n);
  const int end = s == B + 1 ? n : min(max(__ldg(ptr + s), 0), n);
  return make_int2(begin, max(begin, end));
}

// Tile `item` of all scans' tiles of `size` rows (of queries: a row per head of the group); called by one whole warp.
template <bool QUERIES>
__device__ __forceinline__ Work find_work(const Params& p, int item, int size) {
  const int lane = threadIdx.x & 31;
  Work w;
  w.scan = -1;
  int before = 0;
  for (int s0 = 0; s0 < p.B + 2; s0 += 32) {
    const int s = s0 + lane;
    int tiles = 0;
    if (s < p.B + 2) {
      const int2 r = QUERIES ? scan_rows(p.q_ptr, p.B, p.n_q, s) : scan_rows(p.k_ptr, p.B, p.n_k, s);
      const int64_t rows = (int64_t)(r.y - r.x) * (QUERIES ? p.group : 1);
      tiles = (int)((rows + size - 1) / size);
    }
    int upto = tiles;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, upto, o);
      if (lane >= o) upto += v;
    }
    const unsigned here = __ballot_sync(0xffffffffu, before + upto > item);
    if (here) {
      const int l = __ffs((int)here) - 1;
      w.scan = s0 + l;
      w.tile = item - before - (__shfl_sync(0xffffffffu, upto, l) - __shfl_sync(0xffffffffu, tiles, l));
      break;
    }
    before += __shfl_sync(0xffffffffu, upto, 31);
  }
  if (w.scan >= 0) {
    const bool real = w.scan > 0 && w.scan <= p.B;
    const int2 none = make_int2(0, 0);
    const int2 q = real || QUERIES ? scan_rows(p.q_ptr, p.B, p.n_q, w.scan) : none;
    const int2 k = real || !QUERIES ? scan_rows(p.k_ptr, p.B, p.n_k, w.scan) : none;
    w.q0 = q.x; w.nq = q.y - q.x;
    w.k0 = k.x; w.nk = k.y - k.x;
  }
  return w;
}

// Part `split` of `splits` of n rows, in whole tiles of `size`: [first, last).
__device__ __forceinline__ int2 split_rows(int n, int split, int splits, int size) {
  const int per = ((n + size - 1) / size + splits - 1) / splits * size;
  const int first = min((int64_t)n, (int64_t)per * split);
  return make_int2(first, min(n, first + per));
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

inline int most_tiles(int64_t rows, int64_t size, int B) { return (int)(rows / size) + B + 2; }

}  // namespace attn
}  // namespace sph
