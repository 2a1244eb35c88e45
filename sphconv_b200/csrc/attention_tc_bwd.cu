// Gradients of the cross attention on the Blackwell tensor cores (tcgen05), for 16-bit rows of 8 to 128 channels in steps of 8.
//
// One kernel, two directions.  A block has a tile of 128 rows and walks tiles of 64 columns of the other side:
//   KEYS   rows = keys,    columns = queries:  S = K Q^T, dP = V dO^T;  dV += P dO,  dK += dS Q
//   else   rows = queries, columns = keys:     S = Q K^T, dP = dO V^T;               dQ += dS K
//   P = 2^(scale log2 e S - lse),  dS = P (dP - delta);  lse and delta belong to the query: to the column, or to the row.
// Both products of a tile have their A operand in shared memory and give S and dP in TMEM; a thread reads its row of both, writes P and
// dS over them in the rows' type, and these are the A operands of the products behind them, whose B operands are the column
// tiles again, MN-major.  Nothing is transposed, and the accumulators stay in TMEM to the end.  That the scores are made twice, once a
// direction, costs 7 products in place of 5; in return there are no atomics, and results are the same every time.
//
// Warps 0-3: a thread a row; warp 4 issues the MMAs; warps 5-7 copy with cp.async, zeros where there is no row.
//
// float16 has no room below 2^-24: P is held times 2^12, and dS times a power of two of its row's own, that follows its largest value down
// when that outgrows the type (the accumulator is scaled along, as the forward pass does it).
#include <algorithm>

#include "attention_tc.cuh"

namespace sph {
namespace attn {

namespace {

constexpr int kC = 64;                        // columns of a tile
constexpr int kRowWarps = 4, kMmaWarp = 4, kLoadWarp = 5, kLoadWarps = 3;
constexpr int kThreadsTc = (kLoadWarp + kLoadWarps) * 32;
constexpr int kLoaders = kLoadWarps * 32;
constexpr float kShiftP = 12.f;               // fp16: P times 2^12
constexpr float kMostDs = 49152.f, kAimDs = 512.f;    // fp16: dS is scaled to the latter when it would pass the former

template <int DP, bool KEYS>
struct Shape {
  static constexpr bool kWide = DP == 128 && KEYS;          // two wide accumulators: the SM's whole TMEM
  static constexpr int kStages = DP == 128 && !KEYS ? 1 : 2;
  static constexpr uint32_t kRowBytes = (DP / 64) * kM * 128u, kColBytes = (DP / 64) * kC * 128u;
  static constexpr uint32_t kColS = 0, kColDp = 64, kCol1 = 128, kCol2 = KEYS ? 128 + DP : 128;
  static constexpr uint32_t kCols = kWide ? 512 : 256;
  static constexpr int kSmem = 1024 + 2 * (int)kRowBytes + kStages * 2 * (int)kColBytes;
};

template <int DP, bool BF16, bool KEYS>
__global__ void __launch_bounds__(kThreadsTc, 2) backward_tc_kernel(const __grid_constant__ Params p) {
  using S = Shape<DP, KEYS>;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t s_r_full, s_c_full[2], s_c_empty[2], s_stat_full[2], s_s_full, s_p_full, s_done;
  __shared__ __align__(16) float s_lse[2][kC], s_delta[2][kC];
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort;
  __shared__ Work s_work;

  const int tid = threadIdx.x, lane = tid & 31;
  const int warp = (int)uniform((uint32_t)tid >> 5);
  const int split = blockIdx.x % p.splits, rest = blockIdx.x / p.splits;
  const int head = rest % p.hkv, item = rest / p.hkv;
  const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
  const uint32_t r1_at = base, r2_at = base + S::kRowBytes, c_at = base + 2 * S::kRowBytes;      // stage: columns 1, columns 2
  if (tid == 0) {
    s_abort = 0;
    mbar_init(smem_u32(&s_r_full), kLoaders);
    for (int i = 0; i < S::kStages; ++i) {
      mbar_init(smem_u32(&s_c_full[i]), kLoaders);
      mbar_init(smem_u32(&s_c_empty[i]), 1);
      mbar_init(smem_u32(&s_stat_full[i]), kC / 32);
    }
    mbar_init(smem_u32(&s_s_full), 1);
    mbar_init(smem_u32(&s_p_full), kRowWarps);
    mbar_init(smem_u32(&s_done), 1);
    mbar_init_fence();
  }
  after_previous<false>();
  if (warp == 0) {
    const Work w = find_work<!KEYS>(p, item, kM);
    if (lane == 0) s_work = w;
  }
  __syncthreads();
  const Work w = s_work;
  if (w.scan < 0) return;
  const int all = w.nq * p.group;             // rows of queries
  const int2 span = split_rows(KEYS ? all : w.nk, split, p.splits, kC);
  const int tiles = (span.y - span.x + kC - 1) / kC;
  const int row0 = w.tile * kM, rows = min(kM, (KEYS ? w.nk : all) - row0);
  if (warp == kMmaWarp) {
    tmem_alloc(smem_u32(&s_tmem), S::kCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = uniform(s_tmem);
  volatile int* abort_flag = &s_abort;
  // row i of the scan's queries, as a row of [n_q][hq]
  auto query = [&](int i) { return (int64_t)(w.q0 + i / p.group) * p.hq + head * p.group + i % p.group; };

  if (warp < kRowWarps) {
    // ======================= P and dS: thread = row =======================
    const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
    const bool any_row = warp * 32 < rows;
    const bool one = elect_one();
    const int r = warp * 32 + lane;
    const bool mine = r < rows;
    float lse = INFINITY, delta = 0.f;        // of the row
    if (!KEYS && mine) {
      const int64_t at = query(row0 + r);
      lse = p.lse[at];
      delta = p.delta[at];
    }
    float f = 0.f;                            // fp16: dS is held times this; 0: not known yet
    bool dead = false;
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % S::kStages, first = span.x + j * kC, n = min(kC, span.y - first);
      const bool whole = KEYS || (n == kC && p.mask == nullptr);
      uint2 bits = make_uint2(~0u, ~0u);
      if (!whole && any_row) bits = key_bits(p.mask, (int64_t)w.k0 + first, n);
      if (KEYS && !warp_wait(smem_u32(&s_stat_full[st]), (uint32_t)(j / S::kStages) & 1u, abort_flag)) { dead = true; break; }
      if (!warp_wait(smem_u32(&s_s_full), (uint32_t)j & 1u, abort_flag)) { dead = true; break; }
      tc_fence_after();
      if (any_row) {
        // v, u: a piece of the row of S and dP -> P and dS in 32 bits (times 2^12 both, in fp16)
        auto values = [&](int c, uint32_t (&v)[16], uint32_t (&u)[16]) {
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const float l = KEYS ? s_lse[st][c + i] : lse, dl = KEYS ? s_delta[st][c + i] : delta;
            float x = exp2_approx(fmaf(__uint_as_float(v[i]), p.scale_log2, BF16 ? -l : kShiftP - l));
            if (!whole) x = (c < 32 ? bits.x : bits.y) >> ((c & 31) + i) & 1u ? x : 0.f;
            v[i] = __float_as_uint(x);
            u[i] = __float_as_uint(x * (__uint_as_float(u[i]) - dl));
          }
        };
        if (!BF16) {                          // the row's largest dS, and whether it still fits
          float most = 0.f;
#pragma unroll 1
          for (int c = 0; c < kC; c += 16) {
            uint32_t v[16], u[16];
            tmem_ld16(lanes + S::kColS + c, v);
            tmem_ld16(lanes + S::kColDp + c, u);
            tmem_ld_wait();
            values(c, v, u);
#pragma unroll
            for (int i = 0; i < 16; ++i) most = fmaxf(most, fabsf(__uint_as_float(u[i])));
          }
          float by = 1.f;
          if (most > 0.f && (f == 0.f || most * f > kMostDs) && most < INFINITY) {
            // a power of two: exponents only
            const int e = (__float_as_int(kAimDs / most) & 0x7f800000);
            const float now = __int_as_float(min(max(e, 1 << 23), 0x7e800000));
            by = f == 0.f ? 1.f : now / f;
            f = now;
          }
          if (__any_sync(0xffffffffu, by != 1.f) && j > 0) {
#pragma unroll 1
            for (int c = 0; c < p.d; c += 16) {
              uint32_t v[16];
              tmem_ld16(lanes + S::kCol2 + c, v);
              tmem_ld_wait();
#pragma unroll
              for (int i = 0; i < 16; ++i) v[i] = __float_as_uint(__uint_as_float(v[i]) * by);
              tmem_st16(lanes + S::kCol2 + c, v);
            }
          }
        }
        // in the order of columns: P and dS take half of the place of what they are made from
#pragma unroll
        for (int c = 0; c < kC; c += 16) {
          uint32_t v[16], u[16], a[8], b[8];
          tmem_ld16(lanes + S::kColS + c, v);
          tmem_ld16(lanes + S::kColDp + c, u);
          tmem_ld_wait();
          values(c, v, u);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            a[i] = pack2<BF16>(__uint_as_float(v[2 * i]), __uint_as_float(v[2 * i + 1]));
            const float by = BF16 ? 1.f : f;
            b[i] = pack2<BF16>(__uint_as_float(u[2 * i]) * by, __uint_as_float(u[2 * i + 1]) * by);
          }
          if (KEYS) tmem_st8(lanes + S::kColS + c / 2, a);
          tmem_st8(lanes + S::kColDp + c / 2, b);
        }
        tmem_st_wait();
      }
      tc_fence_before();
      __syncwarp();
      if (one) mbar_arrive(smem_u32(&s_p_full));
    }
    // ======================= results =======================
    if (!dead && (tiles == 0 || warp_wait(smem_u32(&s_done), (uint32_t)(tiles - 1) & 1u, abort_flag))) {
      tc_fence_after();
      if (any_row) {
        const bool some = tiles > 0 && mine && (!KEYS || p.mask == nullptr || p.mask[(int64_t)w.k0 + row0 + r] != 0);
        const int64_t of = KEYS ? (int64_t)p.n_k * p.hkv : (int64_t)p.n_q * p.hq;       // rows of a part
        const int64_t at = !mine ? 0 : KEYS ? (int64_t)(w.k0 + row0 + r) * p.hkv + head : query(row0 + r);
        auto store = [&](uint32_t col, float by, void* to, float* part) {
#pragma unroll 1
          for (int c = 0; c < p.d; c += 16) {
            uint32_t v[16];
            tmem_ld16(lanes + col + c, v);
            tmem_ld_wait();
            if (!some) {                      // nothing on the other side, or no key: what the accumulator holds is not looked at
#pragma unroll
              for (int e = 0; e < 16; ++e) v[e] = 0u;
            }
            if (!mine) continue;
            if (p.splits > 1) store16_float(v, by, part + (split * of + at) * p.d + c, p.d - c);
            else store16<BF16>(v, by, (uint16_t*)to + at * p.d + c, p.d - c);
          }
        };
        const float by2 = BF16 ? p.scale : f == 0.f ? p.scale : p.scale * exp2f(-kShiftP) / f;
        store(S::kCol2, by2, KEYS ? p.dk : p.dq, p.part);
        if (KEYS) store(S::kCol1, BF16 ? 1.f : exp2f(-kShiftP), p.dv, p.part2);
      }
    }
  } else if (warp == kMmaWarp) {
    // ======================= MMA issuer =======================
    const bool one = elect_one();
    const uint32_t fmt = BF16 ? 1u : 0u;
    const uint32_t idesc_s = make_idesc(1u, fmt, 0u, 0u, kM, kC);
    const uint32_t idesc_a = make_idesc(1u, fmt, 0u, 1u, kM, (uint32_t)((p.d + 15) / 16 * 16));
    const int steps = (p.d + 15) / 16;        // of 16 channels
    const uint64_t r1 = tile_desc(r1_at, 16u), r2 = tile_desc(r2_at, 16u);
    bool dead = tiles > 0 && !warp_wait(smem_u32(&s_r_full), 0u, abort_flag);
#pragma unroll 1
    for (int j = 0; j < tiles && !dead; ++j) {
      const int st = j % S::kStages;
      const uint32_t c1_at = c_at + st * 2 * S::kColBytes, c2_at = c1_at + S::kColBytes;
      if (!warp_wait(smem_u32(&s_c_full[st]), (uint32_t)(j / S::kStages) & 1u, abort_flag)) break;
      if (j > 0 && !warp_wait(smem_u32(&s_done), (uint32_t)(j - 1) & 1u, abort_flag)) break;      // S goes where P was
      fence_proxy_async();
      tc_fence_after();
      if (one) {
        const uint64_t c1 = tile_desc(c1_at, 16u), c2 = tile_desc(c2_at, 16u);
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
          const uint32_t in = (uint32_t)(s & 3) * 2u;
          umma_f16(tmem + S::kColS, r1 + (s >> 2) * (kM * 8u) + in, c1 + (s >> 2) * (kC * 8u) + in, idesc_s, s ? 1u : 0u);
        }
#pragma unroll 1
        for (int s = 0; s < steps; ++s) {
          const uint32_t in = (uint32_t)(s & 3) * 2u;
          umma_f16(tmem + S::kColDp, r2 + (s >> 2) * (kM * 8u) + in, c2 + (s >> 2) * (kC * 8u) + in, idesc_s, s ? 1u : 0u);
        }
        umma_commit(smem_u32(&s_s_full));
      }
      __syncwarp();
      if (!warp_wait(smem_u32(&s_p_full), (uint32_t)j & 1u, abort_flag)) break;
      tc_fence_after();
      if (one) {
        const uint64_t c1 = tile_desc(c1_at, kC * 128u), c2 = tile_desc(c2_at, kC * 128u);
#pragma unroll
        for (int s = 0; s < kC / 16; ++s) {
          if (KEYS) umma_f16_ta(tmem + S::kCol1, tmem + S::kColS + 8 * s, c2 + (uint64_t)(s * (2048 / 16)), idesc_a, j || s ? 1u : 0u);
          umma_f16_ta(tmem + S::kCol2, tmem + S::kColDp + 8 * s, c1 + (uint64_t)(s * (2048 / 16)), idesc_a, j || s ? 1u : 0u);
        }
        umma_commit(smem_u32(&s_c_empty[st]));
        umma_commit(smem_u32(&s_done));
      }
      __syncwarp();
    }
  } else {
    // ======================= loads =======================
    const int t = tid - kLoadWarp * 32;
    const Pieces pc = pieces_of(p.d);
    const uint8_t* mask = p.mask ? p.mask + w.k0 : nullptr;
    // rows `first` on, n of them, of the queries and of dO, or of keys and values
    auto load_queries = [&](auto size, uint32_t to1, uint32_t to2, int first, int n) {
      constexpr int R = decltype(size)::value;
      load_rows<R, kLoaders>(to1, t, n, p.d, pc, p.q, [&](int r) {
        const int i = first + r;
        return (const uint16_t*)p.q + (int64_t)(w.q0 + i / p.group) * p.q_row + (head * p.group + i % p.group) * p.q_head;
      }, [](int) { return true; });
      load_rows<R, kLoaders>(to2, t, n, p.d, pc, p.d_out, [&](int r) { return (const uint16_t*)p.d_out + query(first + r) * p.d; },
                             [](int) { return true; });
    };
    auto load_keys = [&](auto size, uint32_t to1, uint32_t to2, int first, int n) {
      constexpr int R = decltype(size)::value;
      const uint16_t* k = (const uint16_t*)p.k + (int64_t)(w.k0 + first) * p.k_row + head * p.k_head;
      const uint16_t* v = (const uint16_t*)p.v + (int64_t)(w.k0 + first) * p.v_row + head * p.v_head;
      auto key = [&](int r) { return mask == nullptr || __ldg(mask + first + r) != 0; };
      load_rows<R, kLoaders>(to1, t, n, p.d, pc, p.k, [&](int r) { return k + (int64_t)r * p.k_row; }, key);
      load_rows<R, kLoaders>(to2, t, n, p.d, pc, p.v, [&](int r) { return v + (int64_t)r * p.v_row; }, key);
    };
    using RowTile = std::integral_constant<int, kM>;
    using ColumnTile = std::integral_constant<int, kC>;
    if (tiles > 0) {
      if (KEYS) load_keys(RowTile(), r1_at, r2_at, row0, rows);
      else load_queries(RowTile(), r1_at, r2_at, row0, rows);
      cp_async_arrive_noinc(smem_u32(&s_r_full));
    }
#pragma unroll 1
    for (int j = 0; j < tiles; ++j) {
      const int st = j % S::kStages, first = span.x + j * kC, n = min(kC, span.y - first);
      const uint32_t c1_at = c_at + st * 2 * S::kColBytes;
      if (!warp_wait(smem_u32(&s_c_empty[st]), ((uint32_t)(j / S::kStages) & 1u) ^ 1u, abort_flag)) break;
      if (KEYS) load_queries(ColumnTile(), c1_at, c1_at + S::kColBytes, first, n);
      else load_keys(ColumnTile(), c1_at, c1_at + S::kColBytes, first, n);
      cp_async_arrive_noinc(smem_u32(&s_c_full[st]));
      if (KEYS && t < kC) {
        float lse = INFINITY, delta = 0.f;    // behind the last query: P = 0
        if (t < n) {
          const int64_t at = query(first + t);
          lse = p.lse[at];
          delta = p.delta[at];
        }
        s_lse[st][t] = lse;
        s_delta[st][t] = delta;
        __syncwarp();
        if (lane == 0) mbar_arrive(smem_u32(&s_stat_full[st]));
      }
    }
    cp_async_wait_all();
  }
  tc_fence_before();
  __syncthreads();
  if (s_abort) {
    wind_down(abort_flag, p.status);
    __syncthreads();
  }
  if (warp == kMmaWarp) {
    tc_fence_after();
    tmem_dealloc(tmem, S::kCols);
  }
}

template <int DP, bool BF16, bool KEYS>
int start(const Params& p, int blocks, cudaStream_t st) {
  SPH_CUDA(allow_smem(backward_tc_kernel<DP, BF16, KEYS>, Shape<DP, KEYS>::kSmem));
  launch(backward_tc_kernel<DP, BF16, KEYS>, blocks, kThreadsTc, Shape<DP, KEYS>::kSmem, st, p);
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
int attention_backward_tc_blocks(int d, bool keys) { return d > 64 && keys ? 1 : 2; }       // that share an SM

}  // namespace attn
}  // namespace sph
