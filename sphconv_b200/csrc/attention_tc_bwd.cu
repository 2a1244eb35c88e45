// Gradients of the cross attention on the Blackwell tensor cores (tcgen05), for 16-bit rows of 8 to 128 channels in steps of 8.
//
// One kernel, two directions.  A block has a tile of 128 rows and walks tiles of 64 columns of the other side:
//   KEYS   rows = keys,    columns = queries:  S = K Q^T, dP = V dO^T;  dV += P dO,  dK += dS Q
//   else   rows = queries, columns = keys:     S = Q K^T, dP = dO V^T;               dQ += dS K
//   P = 2^(scale log2 e S - lse),  dS = P (dP - delta);  lse and delta belong to the query: to the column, or to the row.
// Both products of a tile give S and dP in TMEM; a thread reads its row of both, writes P and dS over them in the rows' type, and these
// are the A operands of the products behind them, whose B operands are the column tiles again, MN-major.  Nothing is transposed,
// and the accumulators stay in TMEM to the end.  That the scores are made twice, once a direction, costs 7 products in place of 5 (9 with
// the second value of dS); in return there are no atomics, and results are the same every time.
//
// A block has an SM, with all of its TMEM, and takes one tile of rows after the other: the first scores of the next one are made, and its
// rows brought, while the results of the last are stored.  Warps 0-3 and 4-7 take even and odd tiles of columns, a thread a row; warps 8
// to 11 issue the MMAs of a product each, from waits that do not sleep: S of a place can only be made when the products with the P and
// dS that lay there are complete, and with two or three places (TMEM's room) this chain of handshakes is what a tile takes.  Warps 12 and
// 13 bring columns and rows, by TMA or, where rows are missing or strides unfit, row by row with cp.async, which fills in zeros.
//
// float16 has no room below 2^-24: P is held times 2^15 (its largest is 1; what the rounding of a score in the millions may put on that is
// cut off), and dS times a power of two of its row's own, that follows the row's largest value down when that outgrows the type (the
// accumulator is scaled along).  Even and odd tiles add to one accumulator, so the two warps that have a row take turns at it.
//
// A score's gradients cancel - dS sums to zero over a query's keys - so dS goes into its products as two values of the rows' type, itself and
// what that lost, one product more for either gradient.  P for dV is rounded, and delta comes from the rounded output: with bf16 rows
// dQ is off by 0.0017 to 0.0026 of its size (root mean square), dK by 0.0017 to 0.0019, dV by 0.0024, where their own rounding makes 0.0017.  With dS
// rounded once dQ had 0.0024 to 0.0030 and dK 0.0023 to 0.0027, at 504 us in place of 550:
// 8 scans of 300 queries and 12000 keys, 8 heads of 64 bf16 channels, forward and backward together 550 us; dQ 165, dK and dV 260.  No unit is full:
// with dS rounded once the tensor pipe was 34 and 26 % busy, issue 35 and 44 %.
#include <algorithm>

#include "attention_tc.cuh"

namespace sph {
namespace attn {

namespace {

constexpr int kC = 64;                        // columns of a tile
constexpr int kRowWarps = 8, kScoreWarp = 8, kGradWarp = 10, kColumnWarp = 12;
constexpr int kThreadsTc = 14 * 32;
constexpr float kShiftP = 15.f;               // fp16: P times 2^15
constexpr float kMostDs = 49152.f, kAimDs = 512.f;    // fp16: dS is scaled to the latter when it would pass the former

template <int DP, bool KEYS>
struct Shape {
  static constexpr int kPlaces = DP == 128 && KEYS ? 2 : 3;           // for S and dP
  static constexpr int kStages = DP == 64 ? 4 : 2;                    // of columns
  static constexpr uint32_t kRowBytes = (DP / 64) * kM * 128u, kColBytes = (DP / 64) * kC * 128u;
  static constexpr uint32_t kCol1 = 0, kCol2 = KEYS ? DP : 0, kColS = kCol2 + DP, kCols = 512;
  static __device__ __forceinline__ uint32_t s_at(int b) { return kColS + 128u * b; }
  static __device__ __forceinline__ uint32_t dp_at(int b) { return kColS + 128u * b + 64u; }
  static constexpr int kSmem = 1024 + 4 * (int)kRowBytes + kStages * 2 * (int)kColBytes;      // two tiles of rows
};

// The tensors of a call as maps of 64-row tiles, queries and dO with the heads of a group taken together.
struct Maps {
  TileMap q, d_out, k, v;
};

// P and dS of 16 columns of a row from its S and dP: minus_lse and minus_delta are the row's (4 values alike) or 16 of the columns.
// Times 2^15 both in fp16, which the lse has taken in.
__device__ __forceinline__ void p_and_ds(uint32_t (&v)[16], uint32_t (&u)[16], float scale, const float* minus_lse, const float* minus_delta,
                                         bool columns) {
  const float2 scale2 = make_float2(scale, scale);
#pragma unroll
  for (int i = 0; i < 16; i += 4) {
    const float4 l = *(const float4*)(minus_lse + (columns ? i : 0)), d = *(const float4*)(minus_delta + (columns ? i : 0));
#pragma unroll
    for (int k = 0; k < 4; k += 2) {
      const float2 e = fma2(make_float2(__uint_as_float(v[i + k]), __uint_as_float(v[i + k + 1])), scale2,
                            k ? make_float2(l.z, l.w) : make_float2(l.x, l.y));
      const float2 x = make_float2(exp2_approx(e.x), exp2_approx(e.y));
      const float2 y = mul2(x, add2(make_float2(__uint_as_float(u[i + k]), __uint_as_float(u[i + k + 1])),
                                    k ? make_float2(d.z, d.w) : make_float2(d.x, d.y)));
      v[i + k] = __float_as_uint(x.x); v[i + k + 1] = __float_as_uint(x.y);
      u[i + k] = __float_as_uint(y.x); u[i + k + 1] = __float_as_uint(y.y);
    }
  }
}

// Two values of P; at most 65504 in fp16.
template <bool BF16>
__device__ __forceinline__ uint32_t pack_p(float a, float b) {
  if (BF16) return pack2<BF16>(a, b);
  uint32_t r;
  asm("cvt.rn.satfinite.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(b), "f"(a));
  return r;
}

// One tile of rows against a part of the columns.
struct Item {
  Work w;
  int head, tiles, row0, rows;                // tiles: of columns
};
template <bool KEYS>
__device__ __forceinline__ Item find_item(const Params& p, int index) {          // by whole warps
  Item i;
  i.head = index % p.hkv;
  i.w = find_planned<!KEYS>(p, index / p.hkv);
  i.tiles = i.rows = 0;
  if (i.w.scan < 0) return i;
  i.tiles = (i.w.last - i.w.first + kC - 1) / kC;
  i.row0 = i.w.tile * kM;
  i.rows = (int)min((int64_t)kM, (KEYS ? i.w.nk : (int64_t)i.w.nq * p.group) - i.row0);
  return i;
}

// Where rows of an item's scan lie.
struct Rows {
  const Params& p;
  const Item& i;
  __device__ __forceinline__ int64_t query(int r) const {             // row r of the scan's queries, as a row of [n_q][hq]
    if (p.group == 1) return (int64_t)(i.w.q0 + r) * p.hq + i.head;
    return (int64_t)(i.w.q0 + r / p.group) * p.hq + i.head * p.group + r % p.group;
  }
  __device__ __forceinline__ const uint16_t* q(int r) const {
    if (p.group == 1) return (const uint16_t*)p.q + (int64_t)(i.w.q0 + r) * p.q_row + i.head * p.q_head;
    return (const uint16_t*)p.q + (int64_t)(i.w.q0 + r / p.group) * p.q_row + (i.head * p.group + r % p.group) * p.q_head;
  }
  __device__ __forceinline__ const uint16_t* d_out(int r) const { return (const uint16_t*)p.d_out + query(r) * p.d; }
  __device__ __forceinline__ const uint16_t* k(int r) const { return (const uint16_t*)p.k + (int64_t)(i.w.k0 + r) * p.k_row + i.head * p.k_head; }
  __device__ __forceinline__ const uint16_t* v(int r) const { return (const uint16_t*)p.v + (int64_t)(i.w.k0 + r) * p.v_row + i.head * p.v_head; }
  __device__ __forceinline__ bool is_key(int r) const { return p.mask == nullptr || __ldg(p.mask + (int64_t)i.w.k0 + r) != 0; }
};

// A wait of a whole warp that does not sleep.
__device__ __forceinline__ bool warp_spin(uint32_t bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, mbar_wait_spin(bar, parity, abort_flag));
}

// A wait of a whole warp for as long as a walk may take, which scans of any length have: given up only where `walked`, the tiles that the
// walk has come to, stays as it is for a healthy wait's limit.
__device__ __noinline__ bool wait_for_walk(uint32_t bar, uint32_t parity, volatile int* abort_flag, const volatile int* walked) {
  long long t0 = clock64();
  int before = *walked;
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 64; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, *abort_flag != 0)) return false;
    const int now = *walked;
    if (__any_sync(0xffffffffu, now != before)) {
      before = now;
      t0 = clock64();
    } else if (__any_sync(0xffffffffu, clock64() - t0 > kWaitLimitCycles)) {
      *abort_flag = 1;
      return false;
    }
  }
}

// 64-row boxes of queries and dO (QUERIES), or of keys and values, from row `first` of the scan on, N of them each.
template <int DP, bool QUERIES, int N>
__device__ __forceinline__ void tma_rows(uint32_t to1, uint32_t to2, const Maps& m, const Params& p, const Item& i, int first, uint32_t bar) {
  const int head = QUERIES ? i.head * p.group : i.head;
#pragma unroll
  for (int n = 0; n < N; ++n) {
    const int r = first + 64 * n, at = QUERIES ? i.w.q0 + r / p.group : i.w.k0 + r;
    tma_tile<DP>(to1 + n * 8192u, N * 8192u, QUERIES ? m.q : m.k, head, at, bar);
    tma_tile<DP>(to2 + n * 8192u, N * 8192u, QUERIES ? m.d_out : m.v, head, at, bar);
  }
}

template <int DP, bool BF16, bool KEYS>
__global__ void __launch_bounds__(kThreadsTc, 1) backward_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ Maps m, const int items) {
  using S = Shape<DP, KEYS>;
  constexpr int PL = S::kPlaces, ST = S::kStages;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_r_full[2], s_r_empty[2], s_c_full[ST], s_c_empty[ST], s_s_full[PL], s_p_full[PL], s_done[PL];
  __shared__ __align__(8) uint64_t s_all, s_free, s_some, s_turn[4][2];
  __shared__ __align__(16) float s_stat[kRowWarps][2][kC];  // of a warp's tile: -lse, -delta of the columns
  __shared__ float s_f[2][kM];                // fp16: dS of a row is held times this, of this tile of rows and the last; 0: not known yet
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_walked;           // s_walked: tiles of columns so far

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = (int)uniform((uint32_t)tid >> 5);
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t r_at = base, c_at = base + 4 * S::kRowBytes;         // two operands a tile of rows, and a stage of columns
  constexpr int kGrads = KEYS ? 2 : 1;
  if (tid == 0) {
    s_abort = s_walked = 0;
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_r_full[i]), 1);
      mbar_init(smem_u32(&s_r_empty[i]), 2);
      for (int q = 0; q < 4; ++q) mbar_init(smem_u32(&s_turn[q][i]), 1);
    }
    for (int i = 0; i < ST; ++i) {
      mbar_init(smem_u32(&s_c_full[i]), 1);
      mbar_init(smem_u32(&s_c_empty[i]), kGrads);
    }
    for (int i = 0; i < PL; ++i) {
      mbar_init(smem_u32(&s_s_full[i]), 2);
      mbar_init(smem_u32(&s_p_full[i]), kRowWarps / 2);
      mbar_init(smem_u32(&s_done[i]), kGrads);
    }
    mbar_init(smem_u32(&s_all), kGrads);
    mbar_init(smem_u32(&s_free), kRowWarps);
    mbar_init(smem_u32(&s_some), 1);
    mbar_init_fence();
  }
  if (warp == kScoreWarp) {
    tmem_alloc(smem_u32(&s_tmem), S::kCols);
    tmem_relinquish();
  }
  after_previous<false>();
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(s_tmem);
  volatile int* abort_flag = &s_abort;
  const bool one = elect_one();
  bool dead = false;
  // g counts the tiles of columns since the start, n the tiles of rows that had some
  int g = 0, n = 0;

  if (warp < kRowWarps) {
    // ======================= P and dS: thread = row =======================
    const int half = warp >> 2, quarter = warp & 3;         // half: even or odd tiles
    const uint32_t lanes = tmem + ((uint32_t)(quarter * 32) << 16);
    const int r = quarter * 32 + lane;
    constexpr float kShift = BF16 ? 0.f : kShiftP;
    float *stat_lse = s_stat[warp][0], *stat_delta = s_stat[warp][1];
    float next[4];                            // -lse and -delta of the columns of this warp's next tile: lane and lane + 32
    auto fetch = [&](const Item& it, int j) {
      const Rows at{p, it};
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int c = it.w.first + j * kC + 32 * i + lane;
        const bool some = j < it.tiles && c < it.w.last;
        const int64_t q = some ? at.query(c) : 0;
        next[i] = some ? kShift - p.lse[q] : -INFINITY;
        next[2 + i] = some ? -p.delta[q] : 0.f;
      }
    };
    // tiles alternate between the halves from the start on: the first one of this warp in a tile of rows that g tiles lie in front of
    auto first_tile = [&](int before) { return (before ^ half) & 1; };
    Item it = find_item<KEYS>(p, blockIdx.x), following;
    if (KEYS) fetch(it, first_tile(0));
#pragma unroll 1
    for (int index = blockIdx.x; index < items && !dead; index += gridDim.x, it = following) {
      const Rows at{p, it};
      // what follows is looked for while this one is worked on
      auto look_ahead = [&]() {
        following = find_item<KEYS>(p, index + gridDim.x);
        if (KEYS) fetch(following, first_tile(g + it.tiles));
      };
      if (it.w.scan < 0) {
        look_ahead();
        continue;
      }
      const bool any_row = quarter * 32 < it.rows, mine = r < it.rows;
      float lse = -INFINITY, delta = 0.f;     // minus the row's; -infinity: P = 0
      if (!KEYS && mine) {
        const int64_t q = at.query(it.row0 + r);
        lse = kShift - p.lse[q];
        delta = -p.delta[q];
      }
      // a key, or a query that has some: else its results are zeros, whatever the other side holds
      const bool row_is = mine && (KEYS ? at.is_key(it.row0 + r) : lse != -INFINITY);
      const float row_lse[4] = {lse, lse, lse, lse}, row_delta[4] = {delta, delta, delta, delta};
      const int j0 = first_tile(g);
      float& row_f = s_f[n & 1][r];
#pragma unroll 1
      for (int j = j0; j < it.tiles; j += 2) {
        const int b = (g + j) % PL, k0 = it.w.first + j * kC, cols = min(kC, it.w.last - k0);
        const uint32_t phase = (uint32_t)((g + j) / PL) & 1u;
        const bool whole = KEYS || (cols == kC && p.mask == nullptr);
        uint2 bits = make_uint2(~0u, ~0u);
        if (!whole && any_row) bits = key_bits(p.mask, (int64_t)it.w.k0 + k0, cols);
        if (KEYS) {
          __syncwarp();
          stat_lse[lane] = next[0]; stat_lse[lane + 32] = next[1];
          stat_delta[lane] = next[2]; stat_delta[lane + 32] = next[3];
          __syncwarp();
          fetch(it, j + 2);
        }
        if (!warp_wait(smem_u32(&s_s_full[b]), phase, abort_flag)) { dead = true; break; }
        const uint32_t at_s = lanes + S::s_at(b), at_dp = lanes + S::dp_at(b);
        float f = 1.f;
        auto piece = [&](int c, uint32_t (&v)[16], uint32_t (&u)[16]) {         // 16 columns of P and dS in 32 bits
          tmem_ld16(at_s + c, v);
          tmem_ld16(at_dp + c, u);
          tmem_ld_wait();
          if (!whole) {                       // where there is no key: S -> P = 0, and dP may be anything
            const uint32_t keys = (c < 32 ? bits.x : bits.y) >> (c & 31);
#pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = keys >> i & 1u ? v[i] : 0xff800000u;
          }
          p_and_ds(v, u, p.scale_log2, KEYS ? stat_lse + c : row_lse, KEYS ? stat_delta + c : row_delta, KEYS);
        };
        if (!BF16) {                          // the row's largest dS, and whether it still fits; in the order of the tiles
          float most = 0.f, by = 1.f;
          if (any_row) {
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < kC; c += 16) {
              uint32_t v[16], u[16];
              piece(c, v, u);
#pragma unroll
              for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(__uint_as_float(u[i])));
            }
          }
          // the other warp's turn before: its tile j - 1 is its turn number (g + j - 1) / 2
          if (j > 0 && !warp_wait(smem_u32(&s_turn[quarter][half ^ 1]), (uint32_t)((g + j - 1) >> 1) & 1u, abort_flag)) { dead = true; break; }
          f = j > 0 ? row_f : 0.f;
          if (most > 0.f && (f == 0.f || most * f > kMostDs) && most < INFINITY) {
            // a power of two: exponents only
            const int e = __float_as_int(kAimDs / most) & 0x7f800000;
            const float now = __int_as_float(min(max(e, 1 << 23), 0x7e800000));
            by = f == 0.f ? 1.f : now / f;
            f = now;
          }
          row_f = f;
          if (j > 0 && __any_sync(0xffffffffu, by != 1.f)) {          // behind the tile before, whose dS has the old scale
            const int o = (g + j - 1) % PL;
            if (!warp_wait(smem_u32(&s_done[o]), (uint32_t)((g + j - 1) / PL) & 1u, abort_flag)) { dead = true; break; }
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < p.d; c += 16) {
              uint32_t v[16];
              tmem_ld16(lanes + S::kCol2 + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * by);
              tmem_st16(lanes + S::kCol2 + c, v);
            }
            tmem_st_wait();
            tc_fence_before();
          }
          __syncwarp();
          if (one) mbar_arrive(smem_u32(&s_turn[quarter][half]));
        }
        if (any_row) {
          tc_fence_after();
          // in the order of columns: P and dS take half of the place of what they are made from, and what dS lost in rounding goes
          // where S was (KEYS: to the second half, once that has been read)
          uint32_t lost[kC / 16][8];
#pragma unroll
          for (int c = 0; c < kC; c += 16) {
            uint32_t v[16], u[16], h[8], e[8];
            piece(c, v, u);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              if (KEYS) h[i] = pack_p<BF16>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
              float2 y = make_float2(__uint_as_float(u[2 * i]), __uint_as_float(u[2 * i + 1]));
              if (!BF16) y = mul2(y, make_float2(f, f));
              e[i] = pack2<BF16>(y.x, y.y);
              y = fma2(unpack2<BF16>(e[i]), make_float2(-1.f, -1.f), y);
              lost[c / 16][i] = pack2<BF16>(y.x, y.y);
            }
            if (KEYS) tmem_st8(at_s + c / 2, h);
            tmem_st8(at_dp + c / 2, e);
            if (!KEYS) {
              tmem_st8(at_s + c / 2, lost[c / 16]);
            } else if (c == 32) {
              tmem_st8(at_s + 32, lost[0]);
              tmem_st8(at_s + 40, lost[1]);
            } else if (c == 48) {
              tmem_st8(at_s + 48, lost[2]);
              tmem_st8(at_s + 56, lost[3]);
            }
          }
          tmem_st_wait();
          tc_fence_before();
        }
        __syncwarp();
        if (one) mbar_arrive(smem_u32(&s_p_full[b]));
      }
      // ---- results: KEYS: the first half has dV, the second dK; else each has half of dQ
      look_ahead();
      if (!dead && it.tiles > 0) dead = !warp_wait(smem_u32(&s_all), (uint32_t)n & 1u, abort_flag);
      if (!dead && any_row) {
        tc_fence_after();
        const bool some = it.tiles > 0 && row_is;
        const int64_t of = KEYS ? (int64_t)p.n_k * p.hkv : (int64_t)p.n_q * p.hq;       // rows of a part
        const int64_t to_row = !mine ? 0 : KEYS ? (int64_t)(it.w.k0 + it.row0 + r) * p.hkv + it.head : at.query(it.row0 + r);
        const bool first_of_two = KEYS && half == 0;
        float by = first_of_two ? exp2f(-kShift) : p.scale;
        if (!BF16 && !first_of_two && it.tiles > 0) {
          const int last = g + it.tiles - 1;  // that turn is over, since the products behind it are: this only brings its word
          warp_wait(smem_u32(&s_turn[quarter][last & 1]), (uint32_t)(last >> 1) & 1u, abort_flag);
          const float f = row_f;
          by = f == 0.f ? by : by * exp2f(-kShift) / f;
        }
        const uint32_t col = lanes + (first_of_two ? S::kCol1 : S::kCol2);
        void* to = first_of_two ? p.dv : KEYS ? p.dk : p.dq;
        float* part = first_of_two ? p.part2 : p.part;
#pragma unroll 1
        for (int c = KEYS ? 0 : 16 * half; c < p.d; c += KEYS ? 16 : 32) {
          uint32_t v[16];
          tmem_ld16(col + c, v);
          tmem_ld_wait();
          if (!some) {                        // nothing on the other side, or no key: what the accumulator holds is not looked at
#pragma unroll
            for (int e = 0; e < 16; ++e) v[e] = 0u;
          }
          if (!mine) continue;
          if (p.parts > 1) store16_float(v, by, part + (it.w.part * of + to_row) * p.d + c, p.d - c);
          else store16<BF16>(v, by, (uint16_t*)to + to_row * p.d + c, p.d - c);
        }
        if (mine && p.parts > 1 && it.w.part == 0 && half == 0) p.part_count[to_row] = it.w.parts;
        tc_fence_before();
      }
      __syncwarp();
      if (it.tiles > 0) {
        if (one) mbar_arrive(smem_u32(&s_free));
        ++n;
      }
      g += it.tiles;
    }
  } else if (warp < kColumnWarp) {
    const uint32_t fmt = BF16 ? 1u : 0u;
    const bool columns_fit = KEYS ? m.q.usable && m.d_out.usable : m.k.usable && m.v.usable && p.mask == nullptr;
    if (warp < kGradWarp) {
      // ======================= MMAs of S, and of dP =======================
      const int x = warp - kScoreWarp;
      const uint32_t idesc = make_idesc(1u, fmt, 0u, 0u, kM, kC);
      const int steps = (p.d + 15) / 16;      // of 16 channels
      const uint64_t r_desc = tile_desc(r_at + x * S::kRowBytes, 16u), c_desc = tile_desc(c_at + x * S::kColBytes, 16u);
#pragma unroll 1
      for (int index = blockIdx.x; index < items && !dead; index += gridDim.x) {
        const Item it = find_item<KEYS>(p, index);
        if (it.tiles == 0) continue;
        if (!warp_spin(smem_u32(&s_r_full[n & 1]), (uint32_t)(n >> 1) & 1u, abort_flag)) break;
        fence_proxy_async();
        const uint64_t rows_desc = r_desc + (uint32_t)(n & 1) * (2 * S::kRowBytes / 16u);
#pragma unroll 1
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int st = g % ST, b = g % PL;
          if (!warp_spin(smem_u32(&s_c_full[st]), (uint32_t)(g / ST) & 1u, abort_flag)) { dead = true; break; }
          if (!columns_fit || it.w.last - it.w.first - j * kC < kC) fence_proxy_async();
          if (g >= PL && !warp_spin(smem_u32(&s_done[b]), (uint32_t)((g - PL) / PL) & 1u, abort_flag)) { dead = true; break; }
          tc_fence_after();
          const uint64_t cols_desc = c_desc + (uint32_t)st * (2 * S::kColBytes / 16u);
          const uint32_t to = tmem + (x ? S::dp_at(b) : S::s_at(b));
          if (one) {
#pragma unroll
            for (int s = 0; s < DP / 16; ++s) {
              if (s >= steps) break;
              const int in = (s & 3) * 2, block = s >> 2;
              umma_f16(to, rows_desc + (uint32_t)(block * kM * 8 + in), cols_desc + (uint32_t)(block * kC * 8 + in), idesc, s ? 1u : 0u);
            }
            umma_commit(smem_u32(&s_s_full[b]));
            if (j == it.tiles - 1) umma_commit(smem_u32(&s_r_empty[n & 1]));
          }
        }
        ++n;
      }
    } else if (KEYS || warp == kGradWarp + 1) {
      // ======================= MMAs of the gradients: dV += P dO (KEYS), and dS with Q or K =======================
      const int x = warp - kGradWarp;         // 0: P with the second columns, 1: dS with the first
      const uint32_t idesc = make_idesc(1u, fmt, 0u, 1u, kM, (uint32_t)((p.d + 15) / 16 * 16));
      const uint64_t c_desc = tile_desc(c_at + (x ? 0 : S::kColBytes), kC * 128u);
      const uint32_t to = tmem + (x ? S::kCol2 : S::kCol1);
#pragma unroll 1
      for (int index = blockIdx.x; index < items && !dead; index += gridDim.x) {
        const Item it = find_item<KEYS>(p, index);
        if (it.tiles == 0) continue;
        if (n > 0 && !warp_spin(smem_u32(&s_free), (uint32_t)(n - 1) & 1u, abort_flag)) break;  // the last results have been read
        tc_fence_after();
#pragma unroll 1
        for (int j = 0; j < it.tiles; ++j, ++g) {
          const int st = g % ST, b = g % PL;
          if (!warp_spin(smem_u32(&s_c_full[st]), (uint32_t)(g / ST) & 1u, abort_flag)) { dead = true; break; }
          if (!columns_fit || it.w.last - it.w.first - j * kC < kC) fence_proxy_async();
          if (!warp_spin(smem_u32(&s_p_full[b]), (uint32_t)(g / PL) & 1u, abort_flag)) { dead = true; break; }
          tc_fence_after();
          const uint64_t cols_desc = c_desc + (uint32_t)st * (2 * S::kColBytes / 16u);
          const uint32_t from = tmem + (x ? S::dp_at(b) : S::s_at(b));
          if (one) {
#pragma unroll
            for (int s = 0; s < kC / 16; ++s) umma_f16_ta(to, from + 8 * s, cols_desc + (uint64_t)(s * (2048 / 16)), idesc, j || s ? 1u : 0u);
            if (x) {
#pragma unroll
              for (int s = 0; s < kC / 16; ++s)
                umma_f16_ta(to, tmem + S::s_at(b) + (KEYS ? 32u : 0u) + 8 * s, cols_desc + (uint64_t)(s * (2048 / 16)), idesc, 1u);
            }
            umma_commit(smem_u32(&s_done[b]));
            umma_commit(smem_u32(&s_c_empty[st]));
            if (j == it.tiles - 1) umma_commit(smem_u32(&s_all));
          }
        }
        ++n;
      }
    }
  } else if (warp == kColumnWarp) {
    // ======================= columns =======================
    const Pieces pc = pieces_of(p.d);
    const bool fit = KEYS ? m.q.usable && m.d_out.usable : m.k.usable && m.v.usable && p.mask == nullptr;
    uint32_t ends = 0;                        // tiles with rows missing so far
#pragma unroll 1
    for (int index = blockIdx.x; index < items && !dead; index += gridDim.x) {
      const Item it = find_item<KEYS>(p, index);
      const Rows at{p, it};
#pragma unroll 1
      for (int j = 0; j < it.tiles; ++j, ++g) {
        const int st = g % ST, first = it.w.first + j * kC, cols = min(kC, it.w.last - first);
        const uint32_t to1 = c_at + st * 2 * S::kColBytes, to2 = to1 + S::kColBytes, bar = smem_u32(&s_c_full[st]);
        if (!warp_wait(smem_u32(&s_c_empty[st]), ((uint32_t)(g / ST) & 1u) ^ 1u, abort_flag)) { dead = true; break; }
        if (one) *(volatile int*)&s_walked = g;
        if (fit && cols == kC) {
          if (one) {
            mbar_arrive_expect_tx(bar, 2 * S::kColBytes);
            tma_rows<DP, KEYS, 1>(to1, to2, m, p, it, first, bar);
          }
          continue;
        }
        if (fit) {                            // the scan's last rows: what TMA brought behind them may be anything, and has to be zeros
          const uint32_t some = smem_u32(&s_some);
          if (one) {
            mbar_arrive_expect_tx(some, 2 * S::kColBytes);
            tma_rows<DP, KEYS, 1>(to1, to2, m, p, it, first, some);
          }
          __syncwarp();
          if (!warp_wait(some, ends++ & 1u, abort_flag)) { dead = true; break; }
          const int pieces = (kC - cols) * 8; // of a block of 64 channels: rows are 128 bytes there, in their order
#pragma unroll
          for (int x = 0; x < 2 * (DP / 64); ++x)
            for (int i = lane; i < pieces; i += 32)
              asm volatile("st.shared.v4.b32 [%0], {%1,%1,%1,%1};" ::"r"(to1 + x * (kC * 128u) + (uint32_t)(cols * 128 + i * 16)), "r"(0) : "memory");
          fence_proxy_async();
          __syncwarp();
          if (one) mbar_arrive(bar);
          continue;
        }
        if (KEYS) {
          load_rows<kC, 32>(to1, lane, cols, p.d, pc, p.q, [&](int r) { return at.q(first + r); }, [](int) { return true; });
          load_rows<kC, 32>(to2, lane, cols, p.d, pc, p.d_out, [&](int r) { return at.d_out(first + r); }, [](int) { return true; });
        } else {
          load_rows<kC, 32>(to1, lane, cols, p.d, pc, p.k, [&](int r) { return at.k(first + r); }, [&](int r) { return at.is_key(first + r); });
          load_rows<kC, 32>(to2, lane, cols, p.d, pc, p.v, [&](int r) { return at.v(first + r); }, [&](int r) { return at.is_key(first + r); });
        }
        cp_async_arrive(bar);
        __syncwarp();
        if (one) mbar_arrive(bar);
      }
    }
    cp_async_wait_all();
  } else {
    // ======================= rows: what lies behind the last of them, or in place of a key, is its own row's matter alone =======================
    const Pieces pc = pieces_of(p.d);
    const bool fit = KEYS ? m.k.usable && m.v.usable : m.q.usable && m.d_out.usable;
#pragma unroll 1
    for (int index = blockIdx.x; index < items; index += gridDim.x) {
      const Item it = find_item<KEYS>(p, index);
      if (it.tiles == 0) continue;
      const Rows at{p, it};
      const uint32_t to1 = r_at + (n & 1) * 2 * S::kRowBytes, to2 = to1 + S::kRowBytes, bar = smem_u32(&s_r_full[n & 1]);
      // the tile of rows two before this one keeps its place for all of its walk
      if (!wait_for_walk(smem_u32(&s_r_empty[n & 1]), ((uint32_t)(n >> 1) & 1u) ^ 1u, abort_flag, &s_walked)) break;
      ++n;
      if (fit) {
        if (one) {
          mbar_arrive_expect_tx(bar, 2 * S::kRowBytes);
          tma_rows<DP, !KEYS, 2>(to1, to2, m, p, it, it.row0, bar);
        }
        continue;
      }
      if (KEYS) {
        load_rows<kM, 32>(to1, lane, it.rows, p.d, pc, p.k, [&](int r) { return at.k(it.row0 + r); }, [](int) { return true; });
        load_rows<kM, 32>(to2, lane, it.rows, p.d, pc, p.v, [&](int r) { return at.v(it.row0 + r); }, [](int) { return true; });
      } else {
        load_rows<kM, 32>(to1, lane, it.rows, p.d, pc, p.q, [&](int r) { return at.q(it.row0 + r); }, [](int) { return true; });
        load_rows<kM, 32>(to2, lane, it.rows, p.d, pc, p.d_out, [&](int r) { return at.d_out(it.row0 + r); }, [](int) { return true; });
      }
      cp_async_arrive(bar);
      __syncwarp();
      if (one) mbar_arrive(bar);
    }
    cp_async_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (s_abort) {
    wind_down(abort_flag, p.status);
    __syncthreads();
  }
  if (warp == kScoreWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kCols);
  }
}

template <int DP, bool BF16, bool KEYS>
int start(const Params& p, int blocks, cudaStream_t st) {
  Maps m;
  make_tile_map(&m.q, p.q, p.n_q, p.hq, p.d, p.q_row, p.q_head, kC, p.group);
  make_tile_map(&m.d_out, p.d_out, p.n_q, p.hq, p.d, (int64_t)p.hq * p.d, p.d, kC, p.group);
  make_tile_map(&m.k, p.k, p.n_k, p.hkv, p.d, p.k_row, p.k_head, kC, 1);
  make_tile_map(&m.v, p.v, p.n_k, p.hkv, p.d, p.v_row, p.v_head, kC, 1);
  const int sms = current_sm_count();
  if (sms <= 0) return SPH_ERR_CUDA;
  SPH_CUDA(allow_smem(backward_tc_kernel<DP, BF16, KEYS>, Shape<DP, KEYS>::kSmem));
  launch(backward_tc_kernel<DP, BF16, KEYS>, std::min(blocks, sms), kThreadsTc, Shape<DP, KEYS>::kSmem, st, p, m, blocks);
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}
template <bool KEYS>
int start(const Params& p, bool bf16, int blocks, cudaStream_t st) {
  if (p.d <= 64) return bf16 ? start<64, true, KEYS>(p, blocks, st) : start<64, false, KEYS>(p, blocks, st);
  return bf16 ? start<128, true, KEYS>(p, blocks, st) : start<128, false, KEYS>(p, blocks, st);
}

}  // namespace

int attention_backward_tc(const Params& p, bool bf16, bool keys, int blocks, cudaStream_t st) {
  return keys ? start<true>(p, bf16, blocks, st) : start<false>(p, bf16, blocks, st);
}

}  // namespace attn
}  // namespace sph
