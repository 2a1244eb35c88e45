// What the kernels of the cross attention share: their parameters, and how a block finds its work.
//
// Queries and keys are rows of B scans; scan b has the rows ptr[b] .. ptr[b+1]-1 of each, and what lies in front of the first or behind
// the last scan is treated as two scans more that have nothing on the other side: such rows get zeros.  The lengths are on the device
// only.  A grid has room for as many tiles as any lengths could need, and every block counts through the scans to find its own.
// Where there are few tiles, what each walks over is split into parts: equally long ones, whatever the scans' lengths, as many as the grid
// has room for.  Of a part's results the sums are float32 in a place of their own, and joined in the parts' order by another launch.
//
// Query heads that share a key head are rows of one tile: row r of a scan and key head is query r / group, head r % group.
#pragma once

#include <limits.h>

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
  int parts, aim;                                           // most parts of a tile's walk; how many all tiles are to have about, a head
  float *part, *part2;                                      // with parts > 1: [parts][rows][heads][d], and of dv
  float* part_lse;                                          // forward: [parts][n_q][hq]
  int* part_count;                                          // [rows][heads]
  const struct ScanPlan* plan;                              // [B + 2], where another kernel has left it
  int vec;                                                  // rows can be read in pieces of 16 bytes
  int* status;
};

// Scans that are not in order, or not within the rows, are reported by the first block.
__device__ __forceinline__ void report_scans(const Params& p) {
  if (blockIdx.x != 0 || p.status == nullptr) return;
  bool bad = false;
  for (int b = threadIdx.x; b <= p.B; b += blockDim.x) {
    const int q = __ldg(p.q_ptr + b), k = __ldg(p.k_ptr + b);
    bad |= q < 0 || q > p.n_q || k < 0 || k > p.n_k;
    if (b < p.B) bad |= q > __ldg(p.q_ptr + b + 1) || k > __ldg(p.k_ptr + b + 1);
  }
  if (bad) atomicOr(p.status, SPH_STATUS_BAD_INDEX);
}

// A scan's rows and how they are divided: its tiles' parts are numbers upto - tiles * parts .. upto - 1.
struct __align__(16) ScanPlan {
  int upto, parts, per, tiles;                              // per: rows of the walk that a part has
  int q0, nq, k0, nk;
};

// A tile of queries or keys, and the part of the other side that it is to be walked over with.
struct Work {
  int scan;                                                 // -1: nothing to do
  int tile;
  int q0, nq, k0, nk;                                       // rows of the scan
  int part, parts, first, last;                             // keys, or rows of queries and heads
};

__device__ __forceinline__ int2 scan_rows(const int* ptr, int B, int n, int s) {
  const int begin = s == 0 ? 0 : min(max(__ldg(ptr + s - 1), 0), n);
  const int end = s == B + 1 ? n : min(max(__ldg(ptr + s), 0), n);
  return make_int2(begin, max(begin, end));
}

// Divides the scans' tiles of `size` rows (of queries: a row per head of the group), that are walked over in steps of `step`, into parts;
// by one whole warp, found(plan, first) with 32 scans' plans in its lanes, until it says that this is enough.  A part has `chunk` steps: with
// A steps of all tiles' walks and T tiles, chunk = ceil(A / aim) makes at most aim + T parts.
template <bool QUERIES, typename Found>
__device__ __forceinline__ void plan_scans(const Params& p, int size, int step, Found found) {
  const int lane = threadIdx.x & 31;
  ScanPlan x;
  int steps;
  auto look = [&](int s) {
    int2 q = make_int2(0, 0), k = make_int2(0, 0);
    if (s < p.B + 2) {
      q = scan_rows(p.q_ptr, p.B, p.n_q, s);
      k = scan_rows(p.k_ptr, p.B, p.n_k, s);
      if (s == 0 || s == p.B + 1) (QUERIES ? k : q) = make_int2(0, 0);
    }
    x.q0 = q.x; x.nq = q.y - q.x;
    x.k0 = k.x; x.nk = k.y - k.x;
    const int64_t rows = (int64_t)x.nq * p.group, keys = x.nk;
    x.tiles = (int)(((QUERIES ? rows : keys) + size - 1) / size);
    steps = (int)(((QUERIES ? keys : rows) + step - 1) / step);
  };
  int chunk = INT_MAX;
  if (p.parts > 1) {
    long long a = 0;
    for (int s0 = 0; s0 < p.B + 2; s0 += 32) {
      look(s0 + lane);
      a += (long long)x.tiles * steps;
    }
    for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
    chunk = (int)min(max((a + p.aim - 1) / p.aim, 1ll), (long long)INT_MAX);
  }
  int before = 0;
  for (int s0 = 0; s0 < p.B + 2; s0 += 32) {
    look(s0 + lane);
    const int mine = p.parts > 1 ? max(chunk, (steps + p.parts - 1) / p.parts) : INT_MAX;  // steps of a part
    x.parts = steps == 0 || steps <= mine ? 1 : (steps - 1) / mine + 1;
    x.per = x.parts > 1 ? mine * step : INT_MAX;
    x.upto = x.tiles * x.parts;
    for (int o = 1; o < 32; o <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, x.upto, o);
      if (lane >= o) x.upto += v;
    }
    x.upto += before;
    if (found(x, s0)) break;
    before = __shfl_sync(0xffffffffu, x.upto, 31);
  }
}

// Part `item` as its scan's plan has it.
template <bool QUERIES>
__device__ __forceinline__ Work work_of(const Params& p, const ScanPlan& x, int scan, int item) {
  Work w;
  w.scan = -1;
  const int left = item - (x.upto - x.tiles * x.parts);
  if (left < 0 || left >= x.tiles * x.parts) return w;      // scans that overlap may count up to anything
  w.scan = scan;
  w.parts = x.parts;
  w.tile = x.parts > 1 ? left / x.parts : left;
  w.part = left - w.tile * x.parts;
  w.q0 = x.q0; w.nq = x.nq; w.k0 = x.k0; w.nk = x.nk;
  const int64_t all = QUERIES ? x.nk : (int64_t)x.nq * p.group;
  w.first = (int)min(all, (int64_t)x.per * w.part);
  w.last = (int)min(all, (int64_t)x.per * (w.part + 1));
  return w;
}

// Part `item` of all scans' tiles; by one whole warp.
template <bool QUERIES>
__device__ __forceinline__ Work find_work(const Params& p, int item, int size, int step) {
  Work w;
  w.scan = -1;
  plan_scans<QUERIES>(p, size, step, [&](const ScanPlan& x, int s0) {
    const unsigned here = __ballot_sync(0xffffffffu, x.upto > item);
    if (here == 0) return false;
    const int l = __ffs((int)here) - 1;
    ScanPlan y;
    y.upto = __shfl_sync(0xffffffffu, x.upto, l); y.parts = __shfl_sync(0xffffffffu, x.parts, l);
    y.per = __shfl_sync(0xffffffffu, x.per, l); y.tiles = __shfl_sync(0xffffffffu, x.tiles, l);
    y.q0 = __shfl_sync(0xffffffffu, x.q0, l); y.nq = __shfl_sync(0xffffffffu, x.nq, l);
    y.k0 = __shfl_sync(0xffffffffu, x.k0, l); y.nk = __shfl_sync(0xffffffffu, x.nk, l);
    w = work_of<QUERIES>(p, y, s0 + l, item);
    return true;
  });
  return w;
}
// The same where another kernel has left the plan.
template <bool QUERIES>
__device__ __forceinline__ Work find_planned(const Params& p, int item) {
  const int lane = threadIdx.x & 31;
  Work w;
  w.scan = -1;
  for (int s0 = 0; s0 < p.B + 2; s0 += 32) {
    const int s = s0 + lane;
    const unsigned here = __ballot_sync(0xffffffffu, s < p.B + 2 && __ldg(&p.plan[s].upto) > item);
    if (here == 0) continue;
    const int l = s0 + __ffs((int)here) - 1;
    const int4 a = __ldg((const int4*)(p.plan + l)), b = __ldg((const int4*)(p.plan + l) + 1);
    return work_of<QUERIES>(p, ScanPlan{a.x, a.y, a.z, a.w, b.x, b.y, b.z, b.w}, l, item);
  }
  return w;
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

inline int most_tiles(int64_t rows, int64_t size, int B) { return (int)(rows / size) + B + 2; }

}  // namespace attn
}  // namespace sph
