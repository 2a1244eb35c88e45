// Cross attention on the Blackwell tensor cores (tcgen05), forward, for 16-bit rows of 8 to 128 channels in steps of 8.
//
//   S [128 x 64] = Q K^T    A = a tile of 128 query rows, B = 64 keys, K-major in shared memory; S in TMEM
//   P = 2^(scale log2 e S - top) in the rows' type, written over S by the thread that has the row
//   O [128 x d] += P V      A = P in TMEM, B = the same keys' values, MN-major in shared memory; O stays in TMEM
//
// A block has one tile of queries (heads that share a key head are rows of it) and walks a scan's keys, or a part of them; two blocks
// share an SM.  Keys and values come by TMA where a tile has all of its rows, and row by row with cp.async, which fills in zeros, where
// keys are missing (the scan's end, a mask).
//   bf16: P is taken against the row's maximum in its first tile, without looking for another one: what shows that the maximum has
// grown too far is the sum of P over a tile, above 2^12.  Only then it is searched, O is read, scaled and written again, and P made anew.
// Any P is below 2^12 then, and has all of its bits.
//   float16 has no room for that: it loses bits below 2^-14, and all of them below 2^-25.  Keys far below a row's largest are little each, but tens of
// thousands of them are not, and where their scores are alike so is what each loses (40000 equal ones 16 below one key: the result off by
// 6 %).  So P is held times 2^15, against a maximum that is looked for in every tile and followed when a score is 2^0.9 above it: at most
// 2^-40 of the largest value is lost a key.  200 queries, 8 scans of 87 k rows, 4 heads of 32: 285 us, 248 against the first tile's without the
// factor, 264 with a factor of 2^12 and a maximum that may be 2^3.9 behind.
//
// Warps 0-3 do the softmax, a thread a row; warps 4 and 5 issue the MMAs of S and of O (one warp for both took 1100 cycles a tile, most of
// them waits that were over); warps 6 and 7 load.  S has two places, so that the next scores are there when a row's softmax ends.
// Queries of up to 64 channels are an operand in TMEM: from shared memory, A and B of an MMA of 64 columns take 48 cycles to read and 32
// to multiply.  128 channels leave no columns for them.
//
// P is rounded to the rows' type in front of its product, the sum is of the unrounded ones: a result of bf16 rows is off by 0.0023 of its
// size (root mean square), where its own rounding alone makes 0.0017, of fp16 rows by 0.00027 and 0.00021.  Exponentials are approximate, to
// 2^-22, which is little beside that.
// 4 scans of 2048 queries and 4096 keys, 16 query and 4 key heads of 128 bf16 channels: 233 us, 1180 TFLOP/s, the tensor pipe 56 % busy.
// 8 scans of 256 queries and 87 k keys, 4 heads of 64: 251 us, 730 TFLOP/s; heads of 32: 247 us, of which the exponentials alone, 16 a cycle
// and SM, would take 160.  No unit is full (issue 40 %): what is left is the chain from a tile's scores to its P and back, in two blocks an
// SM.  All eight warps of a block are given 128 registers, of which the four that issue and load need few; moving theirs to the softmax
// warps has not been tried.  Every fourth exponential as a polynomial was slower (267 -> 284 us), and so were tiles of
// 128 keys with one place for S (264 -> 304) and a walk of its own for the maxima (264 -> 334).
#include <algorithm>

#include "attention_tc.cuh"

namespace sph {
namespace attn {

namespace {

constexpr int kN = 64;                        // keys of a tile
constexpr float kMostSum = 4096.f;            // bf16, of a row's P over a tile: above it the row's maximum is taken anew
constexpr float kShiftP = 15.f;               // fp16: P times 2^15
constexpr float kSlack = 0.9f;                // fp16: the row's maximum is taken anew when a score is 2^0.9 above it: 2^15.9 < 65504

// P = 2^(scale s + minus) of N scores in the rows' type, and the sum of P before rounding; fp16: 2^(scale (s + minus) + 15), so that
// the largest score has no rounding to add to its exponent.
template <bool BF16, int N>
__device__ __forceinline__ float row_exp(const uint32_t (&s)[N], uint32_t* h, float scale, float minus) {
  float2 sum[2] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
  const float2 scale2 = make_float2(scale, scale), minus2 = make_float2(minus, minus);
#pragma unroll
  for (int i = 0; i < N; i += 2) {
    const float2 x = make_float2(__uint_as_float(s[i]), __uint_as_float(s[i + 1]));
    const float2 e = BF16 ? fma2(x, scale2, minus2) : fma2(add2(x, minus2), scale2, make_float2(kShiftP, kShiftP));
    const float2 y = make_float2(exp2_approx(e.x), exp2_approx(e.y));
    sum[i / 2 & 1] = add2(sum[i / 2 & 1], y);
    h[i / 2] = pack2<BF16>(y.x, y.y);
  }
  const float2 t = add2(sum[0], sum[1]);
  return t.x + t.y;
}

template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&s)[N]) {
  float most[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
  for (int i = 0; i < N; i += 2) most[i / 2 & 3] = max3(most[i / 2 & 3], __uint_as_float(s[i]), __uint_as_float(s[i + 1]));
  return max3(max3(most[0], most[1], most[2]), most[3], most[3]);
}

// Scores without a key are -infinity.
template <int N>
__device__ __forceinline__ void leave_out(uint32_t (&s)[N], uint32_t keys) {
#pragma unroll
  for (int i = 0; i < N; ++i) s[i] = keys >> i & 1u ? s[i] : 0xff800000u;
}

// A row of O in TMEM times `by`.
__device__ __forceinline__ void scale_row(uint32_t at, int d, float by) {
#pragma unroll 1
  for (int c = 0; c < d; c += 16) {
    uint32_t o[16];
    tmem_ld16(at + c, o);
    tmem_ld_wait();
#pragma unroll
    for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * by);
    tmem_st16(at + c, o);
  }
}

// Row r of a block's tile: of which query and head it is.
struct Row {
  int64_t q;
  int h;
  __device__ __forceinline__ Row(const Params& p, const Work& w, int head, int r) {
    const int i = w.tile * kM + r;
    q = w.q0 + i / p.group;
    h = head * p.group + i % p.group;
  }
  __device__ __forceinline__ const uint16_t* query(const Params& p) const { return (const uint16_t*)p.q + q * p.q_row + h * p.q_head; }
  __device__ __forceinline__ int64_t out(const Params& p) const { return q * p.hq + h; }
};

// The query rows of a tile to shared memory; the warp's arrival included.  Behind the last of them TMA may bring anything: it is a matter
// of its own row's, which is not stored.
template <int DP, int THREADS>
__device__ __forceinline__ void load_queries(uint32_t to, int t, bool first, bool one, int rows, const Params& p, const TileMap& m, const Work& w,
                                             int head, uint32_t bar) {
  if (m.usable) {
    if (one && first) {
      mbar_arrive_expect_tx(bar, DP * kM * 2u);
      tma_tile<DP>(to, kM * 128u, m, head * p.group, w.q0 + w.tile * (kM / p.group), bar);
    } else if (one) {
      mbar_arrive(bar);
    }
    return;
  }
  load_rows<kM, THREADS>(to, t, rows, p.d, pieces_of(p.d), p.q, [&](int r) { return Row(p, w, head, r).query(p); }, [](int) { return true; });
  cp_async_arrive(bar);
  __syncwarp();
  if (one) mbar_arrive(bar);
}

// Whether tile j of a part's keys or values comes by TMA: all of its rows are there.
__device__ __forceinline__ bool by_tma(const Params& p, const TileMap& m, const int2& keys, int j) {
  return m.usable && p.mask == nullptr && keys.y - keys.x - j * kN >= kN;
}

// Tile j of a part's keys, or values, to shared memory, by all loading threads; `first` of their warps issues the TMA loads.
template <int DP, int THREADS>
__device__ __forceinline__ void load_keys(uint32_t to, int t, bool first, bool one, const Params& p, const TileMap& m, const void* x,
                                          int64_t row_stride, int64_t head_stride, const Work& w, const int2& keys, int head, int j,
                                          uint32_t bar) {
  const int at = w.k0 + keys.x + j * kN;
  if (by_tma(p, m, keys, j)) {
    if (one && first) {
      mbar_arrive_expect_tx(bar, DP * kN * 2u);
      tma_tile<DP>(to, kN * 128u, m, head, at, bar);
    } else if (one) {
      mbar_arrive(bar);
    }
    return;
  }
  const uint16_t* from = (const uint16_t*)x + (int64_t)at * row_stride + head * head_stride;
  load_rows<kN, THREADS>(to, t, keys.y - keys.x - j * kN, p.d, pieces_of(p.d), x, [&](int r) { return from + r * row_stride; },
                        [&](int r) { return p.mask == nullptr || __ldg(p.mask + at + r) != 0; });
  cp_async_arrive(bar);
  __syncwarp();
  if (one) mbar_arrive(bar);
}

// S = Q K^T of one tile; by one thread.
template <int DP, bool Q_IN_TMEM>
__device__ __forceinline__ void issue_scores(uint32_t to, uint32_t q_tmem, uint64_t q_desc, uint64_t k_desc, uint32_t idesc, int steps) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    if (s >= steps) break;
    const int in = (s & 3) * 2, block = s >> 2;                       // of a block of 64 channels, in 16 bytes
    const uint64_t k_s = k_desc + (uint32_t)(block * kN * 8 + in);
    if (Q_IN_TMEM) umma_f16_ta(to, q_tmem + 8 * s, k_s, idesc, s ? 1u : 0u);
    else umma_f16(to, q_desc + (uint32_t)(block * kM * 8 + in), k_s, idesc, s ? 1u : 0u);
  }
}
// O += P V of one tile.
__device__ __forceinline__ void issue_out(uint32_t to, uint32_t p_at, uint64_t v_desc, uint32_t idesc, bool first) {
#pragma unroll
  for (int s = 0; s < kN / 16; ++s) umma_f16_ta(to, p_at + 8 * s, v_desc + (uint64_t)(s * (2048 / 16)), idesc, !first || s ? 1u : 0u);
}

// A row's part of the result, from its accumulator at TMEM `at_o`.
template <bool BF16>
__device__ __forceinline__ void store_out(const Params& p, const Work& w, int head, uint32_t at_o, int r, int rows, float top, float sum) {
  const bool none = sum == 0.f, mine = r < rows;
  const int64_t at = Row(p, w, head, min(r, rows - 1)).out(p), part_at = (int64_t)w.part * p.n_q * p.hq + at;
  const float by = none ? 0.f : 1.f / sum, lse = none ? INFINITY : top + log2f(sum);
#pragma unroll 1
  for (int c = 0; c < p.d; c += 16) {
    uint32_t v[16];
    tmem_ld16(at_o + c, v);
    tmem_ld_wait();
    if (none) {                               // no keys: what O holds is not looked at
#pragma unroll
      for (int e = 0; e < 16; ++e) v[e] = 0u;
    }
    if (!mine) continue;
    if (p.parts > 1) store16_float(v, by, p.part + part_at * p.d + c, p.d - c);
    else store16<BF16>(v, by, (uint16_t*)p.out + at * p.d + c, p.d - c);
  }
  if (mine && p.parts > 1 && w.part == 0) p.part_count[at] = w.parts;
  if (mine && p.parts > 1) p.part_lse[part_at] = lse;
  else if (mine && p.lse) p.lse[at] = lse;
}

constexpr int kScoreWarp = 4, kOutWarp = 5, kLoadWarp = 6, kLoadWarps = 2;
constexpr int kThreadsTc = (kLoadWarp + kLoadWarps) * 32, kLoaders = kLoadWarps * 32;

// DP: channels of a tile's rows, 64 or 128.
template <int DP>
struct Shape {
  static constexpr bool kQInTmem = DP == 64;
  static constexpr int kStages = DP == 64 ? 4 : 2;
  static constexpr uint32_t kQBytes = kQInTmem ? 0 : (DP / 64) * kM * 128u, kTileBytes = (DP / 64) * kN * 128u;
  static constexpr uint32_t kColS = 0, kColO = 2 * kN, kColQ = kColO + DP, kCols = 256;
  static constexpr int kSmem = 1024 + (int)kQBytes + 2 * kStages * (int)kTileBytes;
};

template <int DP, bool BF16>
__global__ void __launch_bounds__(kThreadsTc, 2)
forward_tc_kernel(const __grid_constant__ Params p, const __grid_constant__ TileMap q_map, const __grid_constant__ TileMap k_map,
                  const __grid_constant__ TileMap v_map) {
  using S = Shape<DP>;
  constexpr int kStages = S::kStages;
  constexpr uint32_t kTileBytes = S::kTileBytes, kColS = S::kColS, kColO = S::kColO;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_q_full, s_k_full[kStages], s_k_empty[kStages], s_v_full[kStages], s_v_empty[kStages];
  __shared__ __align__(8) uint64_t s_s_full[2], s_p_full[2], s_o_done[2];       // of even and odd tiles
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Work s_work;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = (int)uniform((uint32_t)tid >> 5);
  const int head = blockIdx.x % p.hkv;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t q_at = base, k_at = base + S::kQBytes, v_at = k_at + kStages * kTileBytes;
  if (tid == 0) {
    s_abort = 0;
    mbar_init(smem_u32(&s_q_full), S::kQInTmem ? kScoreWarp : kLoadWarps);
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_u32(&s_k_full[i]), kLoadWarps);
      mbar_init(smem_u32(&s_v_full[i]), kLoadWarps);
      mbar_init(smem_u32(&s_k_empty[i]), 1);
      mbar_init(smem_u32(&s_v_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_u32(&s_s_full[i]), 1);
      mbar_init(smem_u32(&s_p_full[i]), 4);
      mbar_init(smem_u32(&s_o_done[i]), 1);
    }
    mbar_init_fence();
  }
  after_previous<false>();
  report_scans(p);
  if (warp == 0) {
    const Work w = find_work<true>(p, blockIdx.x / p.hkv, kM, kN);
    if (lane == 0) s_work = w;
  }
  __syncthreads();
  const Work w = s_work;
  if (w.scan < 0) return;
  const int2 keys = make_int2(w.first, w.last);
  const int tiles = (keys.y - keys.x + kN - 1) / kN;
  const int rows = min(kM, w.nq * p.group - w.tile * kM);
  if (warp == kScoreWarp) {
    tmem_alloc(smem_u32(&s_tmem), S::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(s_tmem);
  volatile int* abort_flag = &s_abort;

  if (warp < kScoreWarp) {
    // ======================= softmax: thread = row =======================
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const bool any_row = warp * 32 < rows;    // else this warp's lanes hold nothing that is read
    const bool one = elect_one();
    if (S::kQInTmem && tiles > 0) {
      const int r = warp * 32 + lane, pieces = p.d / 8;
      const uint4* from = (const uint4*)Row(p, w, head, min(r, rows - 1)).query(p);
      uint32_t v[32];
#pragma unroll
      for (int c = 0; c < 8; ++c) {
        const uint4 x = r < rows && c < pieces ? __ldg(from + c) : make_uint4(0u, 0u, 0u, 0u);
        v[4 * c] = x.x; v[4 * c + 1] = x.y; v[4 * c + 2] = x.z; v[4 * c + 3] = x.w;
      }
      tmem_st32(lanes + S::kColQ, v);
      tmem_st_wait();
      tc_fence_before();
      __syncwarp();
      if (one) mbar_arrive(smem_u32(&s_q_full));
    }
    float top = -INFINITY, sum = 0.f;         // top: what P is taken against, scaled (fp16: a score as it is)
    bool dead = false;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int first = keys.x + j * kN, n = min(kN, keys.y - first), b = j & 1;
      const bool whole = n == kN && p.mask == nullptr;
      uint2 bits = make_uint2(~0u, ~0u);
      if (!whole && any_row) bits = key_bits(p.mask, (int64_t)w.k0 + first, n);
      if (!warp_wait(smem_u32(&s_s_full[b]), (uint32_t)(j >> 1) & 1u, abort_flag)) { dead = true; break; }
      if (any_row) {
        tc_fence_after();
        uint32_t v[2][kN / 2], h[kN / 2];
        tmem_ld32(lanes + kColS + kN * b, v[0]);
        tmem_ld32(lanes + kColS + kN * b + 32, v[1]);
        tmem_ld_wait();
        if (!whole) {
          leave_out(v[0], bits.x);
          leave_out(v[1], bits.y);
        }
        auto exps = [&]() {                   // where all of the row's scores so far are -infinity, against 0
          const float minus = top == -INFINITY ? 0.f : -top;
          return row_exp<BF16>(v[0], h, p.scale_log2, minus) + row_exp<BF16>(v[1], h + 16, p.scale_log2, minus);
        };
        float add, most;
        bool anew;
        if (BF16) {
          add = exps();
          anew = top == -INFINITY || !(add <= kMostSum);
        } else {
          most = fmaxf(row_max(v[0]), row_max(v[1]));                 // scale > 0
          anew = (most - top) * p.scale_log2 > kSlack;                // NaN where both are infinite: no
        }
        if (__any_sync(0xffffffffu, anew)) {
          float by = 1.f;
          if (BF16) most = fmaxf(row_max(v[0]), row_max(v[1])) * p.scale_log2;
          if (anew && most > top) {
            by = exp2_approx(BF16 ? top - most : (top - most) * p.scale_log2);
            top = most;
            sum *= by;
          }
          if (BF16) add = exps();
          if (j > 0) {
            if (!warp_wait(smem_u32(&s_o_done[b ^ 1]), (uint32_t)((j - 1) >> 1) & 1u, abort_flag)) { dead = true; break; }
            tc_fence_after();
            scale_row(lanes + kColO, p.d, by);
          }
        }
        if (!BF16) add = exps();
        sum += add;
        tmem_st32(lanes + kColS + kN * b, h);
        tmem_st_wait();
        tc_fence_before();
      }
      __syncwarp();
      if (one) mbar_arrive(smem_u32(&s_p_full[b]));
    }
    if (!dead && (tiles == 0 || warp_wait(smem_u32(&s_o_done[(tiles - 1) & 1]), (uint32_t)((tiles - 1) >> 1) & 1u, abort_flag))) {
      tc_fence_after();
      if (any_row) store_out<BF16>(p, w, head, lanes + kColO, warp * 32 + lane, rows, BF16 ? top : fmaf(top, p.scale_log2, -kShiftP), sum);
    }
  } else if (warp == kScoreWarp) {
    // ======================= MMAs of S =======================
    const bool one = elect_one();
    const uint32_t idesc = make_idesc(1u, BF16 ? 1u : 0u, 0u, 0u, kM, kN);
    const int steps = (p.d + 15) / 16;        // of 16 channels
    const uint64_t q_desc = tile_desc(q_at, 16u), k_desc = tile_desc(k_at, 16u);
    bool dead = tiles > 0 && !warp_wait(smem_u32(&s_q_full), 0u, abort_flag);
    if (!S::kQInTmem) fence_proxy_async();
#pragma unroll 1
    for (int j = 0; j < tiles && !dead; ++j) {
      const int st = j % kStages, b = j & 1;
      if (!warp_wait(smem_u32(&s_k_full[st]), (uint32_t)(j / kStages) & 1u, abort_flag)) break;
      if (!by_tma(p, k_map, keys, j)) fence_proxy_async();
      if (j >= 2 && !warp_wait(smem_u32(&s_o_done[b]), (uint32_t)((j - 2) >> 1) & 1u, abort_flag)) break;      // S goes where P was
      tc_fence_after();
      if (one) {
        issue_scores<DP, S::kQInTmem>(tmem + kColS + kN * b, tmem + S::kColQ, q_desc, k_desc + (uint32_t)st * (kTileBytes / 16u), idesc, steps);
        umma_commit(smem_u32(&s_s_full[b]));
        umma_commit(smem_u32(&s_k_empty[st]));
      }
    }
  } else if (warp == kOutWarp) {
    // ======================= MMAs of O =======================
    const bool one = elect_one();
    const uint32_t idesc = make_idesc(1u, BF16 ? 1u : 0u, 0u, 1u, kM, (uint32_t)((p.d + 15) / 16 * 16));
    const uint64_t v_desc = tile_desc(v_at, kN * 128u);
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % kStages, b = j & 1;
      if (!warp_wait(smem_u32(&s_v_full[st]), (uint32_t)(j / kStages) & 1u, abort_flag)) break;
      if (!by_tma(p, v_map, keys, j)) fence_proxy_async();
      if (!warp_wait(smem_u32(&s_p_full[b]), (uint32_t)(j >> 1) & 1u, abort_flag)) break;
      tc_fence_after();
      if (one) {
        issue_out(tmem + kColO, tmem + kColS + kN * b, v_desc + (uint32_t)st * (kTileBytes / 16u), idesc, j == 0);
        umma_commit(smem_u32(&s_o_done[b]));
        umma_commit(smem_u32(&s_v_empty[st]));
      }
    }
  } else {
    // ======================= loads =======================
    const int t = tid - kLoadWarp * 32;
    const bool one = elect_one(), first = warp == kLoadWarp;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % kStages;
      const uint32_t phase = ((uint32_t)(j / kStages) & 1u) ^ 1u;
      if (!warp_wait(smem_u32(&s_k_empty[st]), phase, abort_flag)) break;
      load_keys<DP, kLoaders>(k_at + st * kTileBytes, t, first, one, p, k_map, p.k, p.k_row, p.k_head, w, keys, head, j,
                               smem_u32(&s_k_full[st]));
      if (!S::kQInTmem && j == 0)
        load_queries<DP, kLoaders>(q_at, t, first, one, rows, p, q_map, w, head, smem_u32(&s_q_full));      // behind the first keys
      if (!warp_wait(smem_u32(&s_v_empty[st]), phase, abort_flag)) break;
      load_keys<DP, kLoaders>(v_at + st * kTileBytes, t, first, one, p, v_map, p.v, p.v_row, p.v_head, w, keys, head, j,
                               smem_u32(&s_v_full[st]));
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

template <int DP, bool BF16>
int start(const Params& p, int blocks, cudaStream_t st) {
  TileMap q_map, k_map, v_map;
  make_tile_map(&q_map, p.q, p.n_q, p.hq, p.d, p.q_row, p.q_head, kM, p.group);
  make_tile_map(&k_map, p.k, p.n_k, p.hkv, p.d, p.k_row, p.k_head, kN, 1);
  make_tile_map(&v_map, p.v, p.n_k, p.hkv, p.d, p.v_row, p.v_head, kN, 1);
  SPH_CUDA(allow_smem(forward_tc_kernel<DP, BF16>, Shape<DP>::kSmem));
  launch(forward_tc_kernel<DP, BF16>, blocks, kThreadsTc, Shape<DP>::kSmem, st, p, q_map, k_map, v_map);
  SPH_LAUNCH_CHECK();
  return SPH_OK;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                 const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                 CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
EncodeTiled encode_tiled() {
  static const EncodeTiled fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult found;
    if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &f, 12000, cudaEnableDefault, &found) != cudaSuccess ||
        found != cudaDriverEntryPointSuccess)
      f = nullptr;
    return (EncodeTiled)f;
  }();
  return fn;
}

}  // namespace

void make_tile_map(TileMap* m, const void* x, int64_t rows, int heads, int d, int64_t row_stride, int64_t head_stride, int tile, int group) {
  *m = TileMap{};
  const EncodeTiled encode = encode_tiled();
  if (encode == nullptr || rows < 1 || tile % group != 0) return;
  // a dimension of one entry has any stride
  const int64_t hs = heads > 1 ? head_stride * 2 : 128, rs = rows > 1 ? row_stride * 2 : 128;
  if (hs <= 0 || rs <= 0 || hs % 16 != 0 || rs % 16 != 0 || ((uintptr_t)x & 15) != 0) return;
  m->rows_inside = group == 1 && hs > rs;
  const bool in = m->rows_inside;
  const cuuint64_t dims[3] = {(cuuint64_t)d, (cuuint64_t)(in ? rows : heads), (cuuint64_t)(in ? heads : rows)};
  const cuuint64_t strides[2] = {(cuuint64_t)(in ? rs : hs), (cuuint64_t)(in ? hs : rs)};
  const cuuint32_t box[3] = {64, (cuuint32_t)(in ? tile : group), (cuuint32_t)(in ? 1 : tile / group)}, steps[3] = {1, 1, 1};
  m->usable = encode(&m->map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 3, const_cast<void*>(x), dims, strides, box, steps,
                     CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

int attention_forward_tc(const Params& p, bool bf16, int blocks, cudaStream_t st) {
  if (p.d <= 64) return bf16 ? start<64, true>(p, blocks, st) : start<64, false>(p, blocks, st);
  return bf16 ? start<128, true>(p, blocks, st) : start<128, false>(p, blocks, st);
}

}  // namespace attn
}  // namespace sph
