// The products x = h W^T of the log-probability entries, whose logits never leave the SM: a tcgen05
// kernel on CTA pairs (256 x 256 tiles, cta_group::2, operands by TMA, accumulators double-buffered in
// tensor memory) with two epilogues.
//
// LP_STATS keeps, for each row, the running maximum, sum of exponentials and entropy sum of the softmax in
// registers from tile to tile, and the best K logits in a sorted register list: an epilogue thread owns
// half of a row's columns. A chunk of 32 logits costs its maximum and four instructions a logit; only
// where the maximum beats the K-th best so far (about K ln(V / K) times a row) the warp looks for the
// logits that do, reading them once more from tensor memory.
// LP_GRAD writes the logits' gradient ([v = t] a - p (a + b (log p + H))) in the operand type of the
// products that follow.
//
// Each CTA pair takes one run of consecutive tiles, all of the same length to within one, in an order
// that keeps a row block until its columns are done: h's tile and the rows' state stay, W streams from
// L2. (One column group at a time where W does not fit there.) So all pairs end together whatever N and
// V are, and a row block is cut into at most `slots` shares, which lp_join_kernel adds up.
//
// fp32 operands are given as three bf16 parts each (x = hi + mid + lo to the last bit, lp_split_kernel),
// and the product runs over six pairs of parts, the small ones first: what is left out is below 2^-25 of
// each product. Bound by the tensor cores either way.
#include <algorithm>

#include "gemm.cuh"

namespace ulm {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int LP_MAX_TOP = 32;  // top_k of the entries

enum { LP_STATS = 0, LP_GRAD = 1 };
constexpr int LPM_STAGES = 5;
constexpr int LPM_SLOTS = 2;  // 4 KB staging tiles of an epilogue warp (LP_GRAD)
constexpr uint32_t LPM_HALF_BYTES = 128 * 64 * 2;  // a CTA's 128 rows of one operand, 64 k values
constexpr uint32_t LPM_STAGE_BYTES = 2 * LPM_HALF_BYTES;
constexpr uint32_t LPM_SMEM = LPM_STAGES * LPM_STAGE_BYTES + EPI_WARPS * LPM_SLOTS * 4096u + 1024 + 512;
static_assert(LPM_SMEM <= 232448, "shared memory of one CTA");

// The shape of a launch; total tiles are dealt to `pairs` CTA pairs, pair p the run [first(p), first(p + 1)).
struct LpShape {
  int N, V;
  int kblocks;           // 64-wide k blocks of one pair of parts
  int parts;             // pairs of operand parts: 1, or 6 for fp32 operands
  int row_blocks, col_tiles, group;  // group: column tiles done for all rows before the next ones
  int pairs, slots;      // slots: shares that a row block can have in one column group
  int64_t total;
};

struct LpTile {
  int rb, ct, g;  // row block, column tile, column group
};
__host__ __device__ inline int64_t lp_first(const LpShape& s, int p) { return p * s.total / s.pairs; }
__host__ __device__ inline int lp_pair_of(const LpShape& s, int64_t t) { return (int)(((t + 1) * s.pairs - 1) / s.total); }
// first tile of row block rb in column group g
__host__ __device__ inline int64_t lp_row_first(const LpShape& s, int g, int rb) {
  const int rest = s.col_tiles - g * s.group;
  return (int64_t)g * s.group * s.row_blocks + (int64_t)rb * (rest < s.group ? rest : s.group);
}
__device__ __forceinline__ LpTile lp_tile(const LpShape& s, int64_t t) {
  const int64_t per_group = (int64_t)s.group * s.row_blocks;
  LpTile r;
  r.g = (int)(t / per_group);
  const int rem = (int)(t - r.g * per_group);
  const int wide = min(s.group, s.col_tiles - r.g * s.group);
  r.rb = rem / wide;
  r.ct = r.g * s.group + rem - r.rb * wide;
  return r;
}

// What an epilogue reads and writes.
struct LpArgs {
  const int64_t* tokens;
  // LP_STATS: for share i = ((row * groups + g) * slots + slot) * 2 + half of a row: (max, sum, entropy sum)
  // in part[4 i] (base 2: of 2^(x log2 e - max log2 e)), its best logits in list[i * K] as (value, id), and
  // given[row], the token's logit
  float* part;
  float2* list;
  float* given;
  int groups;
  // LP_GRAD
  const float* stats;
  const float* entropy;
  const float* dlogprobs;
  const float* dentropy;
};

__device__ __forceinline__ void tmem_ld_32x1(uint32_t taddr, float& x) {
  uint32_t r;
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];\n\ttcgen05.wait::ld.sync.aligned;"
               : "=r"(r)
               : "r"(taddr)
               : "memory");
  x = __uint_as_float(r);
}

// The backward's factors of one row: dx_v = ([v = t] a) - p_v (a + b (log p_v + H)).
struct LpCoef {
  float base, logs, c0, b, a;
  int64_t t;
};
__device__ __forceinline__ LpCoef lp_coef(const int64_t* tokens, const float* stats, const float* entropy,
                                          const float* dlogprobs, const float* dentropy, int64_t r, int V) {
  LpCoef c;
  c.t = tokens[r];
  c.base = stats[2 * r];
  c.logs = stats[2 * r + 1];
  c.a = c.t == -1 || !dlogprobs ? 0.f : dlogprobs[r];
  if (c.t < -1 || c.t >= V) c.a = __uint_as_float(0x7FC00000u);
  c.b = dentropy ? dentropy[r] : 0.f;
  c.c0 = c.a + (c.b != 0.f ? c.b * entropy[r] : 0.f);
  return c;
}

// The statistics of one thread's share of a row, over chunks of 32 logits.
template <int K>
struct LpRun {
  float m, m2, s, u;  // maximum (at least -1e30), m log2 e, sum 2^(x log2 e - m2), sum 2^(.) (.)
  float v[K > 0 ? K : 1];
  int id[K > 0 ? K : 1];

  __device__ __forceinline__ void reset(bool live) {
    m = -1e30f;
    m2 = m * LOG2E;
    s = u = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j] = live ? -INFINITY : INFINITY;  // nothing beats the list of a row that is not there
      id[j] = -1;
    }
  }
  __device__ __forceinline__ void insert(float x, int i) {
#pragma unroll
    for (int j = K - 1; j > 0; --j) {
      const bool up = x > v[j - 1], here = x > v[j];
      v[j] = up ? v[j - 1] : here ? x : v[j];
      id[j] = up ? id[j - 1] : here ? i : id[j];
    }
    if (x > v[0]) {
      v[0] = x;
      id[0] = i;
    }
  }
  // logits of columns col0 .. col0 + 31 (in tensor memory at taddr), V the first column past the last
  __device__ __forceinline__ void add(const uint32_t (&r)[32], uint32_t taddr, int col0, int V) {
    float x[32];
#pragma unroll
    for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
    if (col0 + 32 > V) {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = col0 + i < V ? x[i] : -1e30f;
    }
    float lm = fmaxf(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 32; i += 2) lm = fmaxf(lm, fmaxf(x[i], x[i + 1]));
    if (lm > m) {
      const float n2 = lm * LOG2E, d = m2 - n2, f = fast_exp2(d);
      u = f > 0.f ? (u + s * d) * f : 0.f;
      s *= f;
      m = lm;
      m2 = n2;
    }
    float s0 = 0.f, s1 = 0.f, u0 = 0.f, u1 = 0.f;
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const float d0 = fmaf(x[i], LOG2E, -m2), d1 = fmaf(x[i + 1], LOG2E, -m2);
      const float e0 = fast_exp2(d0), e1 = fast_exp2(d1);
      s0 += e0;
      s1 += e1;
      u0 = fmaf(e0, d0, u0);
      u1 = fmaf(e1, d1, u1);
    }
    s += s0 + s1;
    u += u0 + u1;
    if (K > 0) {
      if (__any_sync(0xffffffffu, lm > v[K - 1])) {
        uint32_t bits = 0;
#pragma unroll
        for (int i = 0; i < 32; ++i) bits |= x[i] > v[K - 1] ? 1u << i : 0u;
        bits = __reduce_or_sync(0xffffffffu, bits);
        while (bits) {
          const int i = __ffs(bits) - 1;
          bits &= bits - 1;
          float y;
          tmem_ld_32x1(taddr + (uint32_t)i, y);
          if (y > v[K - 1] && col0 + i < V) insert(y, col0 + i);
          __syncwarp();
        }
      }
    }
  }
};

template <int MODE, int K, bool F32>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(TC_THREADS, 1)
    lp_mma_kernel(const __grid_constant__ CUtensorMap tma_h, const __grid_constant__ CUtensorMap tma_w,
                  const __grid_constant__ CUtensorMap tma_out, const LpShape shape, const LpArgs args) {
  constexpr int STAGES = LPM_STAGES;
  constexpr uint32_t IDESC = idesc_bf16_f32(256, 256, false, false);
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* stage_out = smem + STAGES * LPM_STAGE_BYTES;
  uint64_t* full = reinterpret_cast<uint64_t*>(stage_out + EPI_WARPS * LPM_SLOTS * 4096u);
  uint64_t* empty = full + STAGES;
  uint64_t* tfull = empty + STAGES;
  uint64_t* tempty = tfull + 2;
  uint64_t* drain = tempty + 2;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(drain + 1);
  volatile int* abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);

  const int warp = threadIdx.x >> 5;
  const int lane = threadIdx.x & 31;
  const uint32_t rank = cluster_ctarank();
  const bool leader = rank == 0;
  const int pair = blockIdx.x >> 1;
  const int64_t t_first = lp_first(shape, pair), t_end = lp_first(shape, pair + 1);

  if (threadIdx.x == 0) {
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&tfull[a], 1);
      mbar_init(&tempty[a], 2 * EPI_WARPS);  // the epilogue warps of both CTAs
    }
    mbar_init(drain, 1);
    *abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == 0 && lane == 0) {
    tma_prefetch_desc(&tma_h);
    tma_prefetch_desc(&tma_w);
    if (MODE == LP_GRAD) tma_prefetch_desc(&tma_out);
  }
  if (warp == 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_slot;
  pdl_enter();

  if (warp == 0) {
    if (lane == 0) {
      // ---------------- producer (both CTAs): 128 rows of h and of W for each k block ----------------
      const uint32_t leader_full = mapa_shared(smem_u32(full), 0);
      int stage = 0;
      uint32_t phase = 0;
      int issued = 0;
      bool ok = true;
      for (int64_t t = t_first; t < t_end && ok; ++t) {
        const LpTile tile = lp_tile(shape, t);
        const int row0 = tile.rb * 256 + (int)rank * 128, col0 = tile.ct * 256 + (int)rank * 128;
        for (int q = 0; q < shape.parts && ok; ++q) {
          const int ph = shape.parts > 1 ? GEMM_PART_A[q] : 0, pw = shape.parts > 1 ? GEMM_PART_B[q] : 0;
          for (int kb = 0; kb < shape.kblocks; ++kb) {
            if (!wait_or_abort(&empty[stage], phase ^ 1u, abort_flag, DEVERR_LOGPROBS_WAIT)) {
              ok = false;
              break;
            }
            uint8_t* sa = smem + stage * LPM_STAGE_BYTES;
            const uint32_t bar = leader_full + (uint32_t)(stage * sizeof(uint64_t));
            if (leader) mbar_arrive_expect_tx(&full[stage], 2 * LPM_STAGE_BYTES);
            tma_load_3d_pair(&tma_h, sa, bar, kb * 64, row0, ph);
            tma_load_3d_pair(&tma_w, sa + LPM_HALF_BYTES, bar, kb * 64, col0, pw);
            issued = min(issued + 1, STAGES);
            if (++stage == STAGES) {
              stage = 0;
              phase ^= 1u;
            }
          }
        }
      }
      if (!ok && leader) {
        // drain: wait (bounded) for the loads still in flight
        for (int i = 0; i < issued; ++i) {
          if (--stage < 0) {
            stage = STAGES - 1;
            phase ^= 1u;
          }
          const uint64_t t0 = globaltimer_ns();
          while (!mbar_try_wait(&full[stage], phase) && globaltimer_ns() - t0 < 100000000ull) {
          }
        }
      }
    }
  } else if (warp == 1) {
    if (lane == 0 && leader) {
      // ---------------- MMA issuer (leader CTA) ----------------
      int stage = 0;
      uint32_t phase = 0;
      int j = 0;
      bool ok = true, issued_any = false;
      const int nkb = shape.parts * shape.kblocks;
      for (int64_t t = t_first; t < t_end && ok; ++t, ++j) {
        const int acc = j & 1;
        if (!wait_or_abort(&tempty[acc], ((uint32_t)(j >> 1) & 1u) ^ 1u, abort_flag, DEVERR_LOGPROBS_WAIT)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t d_tmem = tmem_base + (uint32_t)(acc * 256);
        for (int i = 0; i < nkb; ++i) {
          if (!wait_or_abort(&full[stage], phase, abort_flag, DEVERR_LOGPROBS_WAIT)) {
            ok = false;
            break;
          }
          tc_fence_after();
          const uint32_t sa = smem_u32(smem + stage * LPM_STAGE_BYTES);
          const uint32_t sb = sa + LPM_HALF_BYTES;
#pragma unroll
          for (int kk = 0; kk < 4; ++kk)
            umma_bf16_ss_pair(d_tmem, smem_desc_sw128(sa + kk * 32, 16, 1024), smem_desc_sw128(sb + kk * 32, 16, 1024),
                              IDESC, (i > 0 || kk > 0) ? 1u : 0u);
          issued_any = true;
          umma_commit_pair(&empty[stage], 0x3);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
        if (!ok) break;
        umma_commit_pair(&tfull[acc], 0x3);
      }
      if (!ok && issued_any) {
        umma_commit_pair(drain, 0x1);
        const uint64_t t0 = globaltimer_ns();
        while (!mbar_try_wait(drain, 0) && globaltimer_ns() - t0 < 100000000ull) {
        }
      }
    }
  } else {
    // ---------------- epilogue: warp w has TMEM lane quadrant w % 4 and 128 of the tile's columns ------
    const int ew = warp - 2, quad = warp & 3, half = ew >> 2;
    const uint32_t leader_tempty = mapa_shared(smem_u32(tempty), 0);
    uint8_t* slots = stage_out + ew * (LPM_SLOTS * 4096);
    int n = 0;  // staged chunks so far
    int j = 0;
    int at_g = -1, at_rb = -1;
    int64_t row = 0, tok = -1;
    bool live = false;
    LpRun<K> run;
    LpCoef c;
    if (MODE == LP_STATS) run.reset(false);
    auto flush = [&]() {
      if (MODE != LP_STATS || at_rb < 0 || !live) return;
      const int slot = pair - lp_pair_of(shape, lp_row_first(shape, at_g, at_rb));
      const int64_t i = ((row * args.groups + at_g) * shape.slots + slot) * 2 + half;
      *reinterpret_cast<float4*>(args.part + 4 * i) = make_float4(run.m, run.s, run.u, 0.f);
      if (K > 0) {
#pragma unroll
        for (int q = 0; q < K; ++q) args.list[i * K + q] = make_float2(run.v[q], __int_as_float(run.id[q]));
      }
    };
    for (int64_t t = t_first; t < t_end; ++t, ++j) {
      const LpTile tile = lp_tile(shape, t);
      if (tile.rb != at_rb || tile.g != at_g) {
        flush();
        at_rb = tile.rb;
        at_g = tile.g;
        row = (int64_t)tile.rb * 256 + (int64_t)rank * 128 + quad * 32 + lane;
        live = row < shape.N;
        if (MODE == LP_STATS) {
          run.reset(live);
          tok = live ? args.tokens[row] : -1;
        } else {
          c = live ? lp_coef(args.tokens, args.stats, args.entropy, args.dlogprobs, args.dentropy, row, shape.V)
                   : LpCoef{0.f, 0.f, 0.f, 0.f, 0.f, -1};
          tok = c.t;
        }
      }
      const int acc = j & 1;
      if (!wait_or_abort(&tfull[acc], (uint32_t)(j >> 1) & 1u, abort_flag, DEVERR_LOGPROBS_WAIT)) break;
      tc_fence_after();
      const uint32_t taddr = tmem_base + ((uint32_t)(quad * 32) << 16) + (uint32_t)(acc * 256 + half * 128);
      const int col_base = tile.ct * 256 + half * 128;
      const bool rows_here = __any_sync(0xffffffffu, live);
      const int chunks = rows_here ? min(4, (shape.V - col_base + 31) / 32) : 0;
      if (MODE == LP_STATS) {
        uint32_t ra[32], rb[32];
        if (chunks > 0) tmem_ld_32x32_issue(taddr, ra);
        auto one = [&](const uint32_t(&r)[32], int ch) {
          const int col0 = col_base + 32 * ch;
          run.add(r, taddr + (uint32_t)(32 * ch), col0, shape.V);
          if (tok >= col0 && tok < col0 + 32 && tok < shape.V) {
            float g = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col0 + i == (int)tok) g = __uint_as_float(r[i]);
            args.given[row] = g;
          }
          __syncwarp();
        };
#pragma unroll
        for (int ch = 0; ch < 4; ch += 2) {
          if (ch < chunks) {
            tmem_ld_32x32_wait(ra);
            if (ch + 1 < chunks) tmem_ld_32x32_issue(taddr + 32 * (ch + 1), rb);
            one(ra, ch);
          }
          if (ch + 1 < chunks) {
            tmem_ld_32x32_wait(rb);
            if (ch + 2 < chunks) tmem_ld_32x32_issue(taddr + 32 * (ch + 2), ra);
            one(rb, ch + 1);
          }
        }
      } else {
        constexpr int CW = F32 ? 32 : 64;  // columns of a staged chunk of 128 bytes a row
        const int nch = rows_here ? min(128 / CW, (shape.V - col_base + CW - 1) / CW) : 0;
#pragma unroll 1
        for (int i = 0; i < nch; ++i) {
          uint8_t* out = slots + (n % LPM_SLOTS) * 4096;
          ++n;
          if (lane == 0) bulk_wait_group_read<LPM_SLOTS - 1>();  // the store before last has read its slot
          __syncwarp();
#pragma unroll
          for (int hh = 0; hh < CW / 32; ++hh) {
            float v[32];
            const int col0 = col_base + i * CW + hh * 32;
            tmem_ld_32x32(taddr + (uint32_t)(i * CW + hh * 32), v);
#pragma unroll
            for (int q = 0; q < 32; ++q) {
              const float logp = (v[q] - c.base) - c.logs;
              v[q] = -fast_exp2(logp * LOG2E) * fmaf(c.b, logp, c.c0);
            }
            if (tok >= col0 && tok < col0 + 32) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (col0 + q == (int)tok) v[q] += c.a;
            }
            __syncwarp();
            stage_write<F32, 32>(out, lane, hh * (F32 ? 8 : 4), v);
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            tma_store_3d(&tma_out, out, col_base + i * CW, tile.rb * 256 + (int)rank * 128 + quad * 32, 0);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster(leader_tempty + (uint32_t)(acc * sizeof(uint64_t)));
    }
    flush();
    if (MODE == LP_GRAD && lane == 0) bulk_wait_group<0>();
  }

  tc_fence_before();
  cluster_sync_all();  // all MMAs done and all TMEM reads finished in both CTAs
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// One warp per row: its shares' statistics merged, its K-lists merged by k rounds of the best remaining
// head (value descending, id ascending). Each lane keeps the heads of every 32nd list.
__global__ void __launch_bounds__(128)
    lp_join_kernel(const LpShape shape, const LpArgs args, int K, float* __restrict__ logprobs,
                   float* __restrict__ entropy, float* __restrict__ stats, int64_t* __restrict__ top_ids,
                   float* __restrict__ top_logprobs, int k) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= shape.N) return;
  const int rb = (int)(row / 256);
  const int all = args.groups * shape.slots * 2;  // the row's possible shares
  // whether share i is there: its pair took tiles of this row block
  auto there = [&](int i) {
    const int g = i / (2 * shape.slots), slot = (i / 2) % shape.slots;
    const int64_t a = lp_row_first(shape, g, rb), b = a + min(shape.group, shape.col_tiles - g * shape.group);
    return lp_pair_of(shape, a) + slot <= lp_pair_of(shape, b - 1);
  };
  uint32_t mine = 0;  // bit j: share lane + 32 j is there
  for (int j = 0; 32 * j + lane < all; ++j) mine |= there(32 * j + lane) ? 1u << j : 0u;
  const float4* part = reinterpret_cast<const float4*>(args.part) + row * all;
  float m = -1e30f;
  for (int i = lane, j = 0; i < all; i += 32, ++j)
    if ((mine >> j) & 1u) m = fmaxf(m, part[i].x);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
  const float m2 = m * LOG2E;
  float s = 0.f, u = 0.f;
  for (int i = lane, j = 0; i < all; i += 32, ++j)
    if ((mine >> j) & 1u) {
      const float4 p = part[i];
      const float d = p.x * LOG2E - m2, f = fast_exp2(d);
      s = fmaf(p.y, f, s);
      if (f > 0.f) u += (p.z + p.y * d) * f;
    }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    s += __shfl_xor_sync(0xffffffffu, s, o);
    u += __shfl_xor_sync(0xffffffffu, u, o);
  }
  // logp = (x - m) - logs with log s + (m2 ln 2 - m), the second term the rounding of m2
  const float logs = logf(s) + fmaf(LN2, m2, -m);
  if (lane == 0) {
    const int64_t t = args.tokens[row];
    logprobs[row] = t == -1 ? 0.f : t < 0 || t >= shape.V ? __uint_as_float(0x7FC00000u) : (args.given[row] - m) - logs;
    entropy[row] = logf(s) - LN2 * (u / s);
    if (stats) {
      stats[2 * row] = m;
      stats[2 * row + 1] = logs;
    }
  }
  if (k == 0) return;
  const float2* list = args.list + row * all * K;
  uint32_t used[8];  // how many of each of its lists' entries a lane has given, 8 bits each
#pragma unroll
  for (int i = 0; i < 8; ++i) used[i] = 0;
  for (int r = 0; r < k; ++r) {
    float bv = -INFINITY;
    int bid = 0x7fffffff, bl = -1;
#pragma unroll
    for (int w = 0; w < 8; ++w)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int i = lane + 32 * (4 * w + q);
        if ((mine >> (4 * w + q)) & 1u) {
          const int at = (used[w] >> (8 * q)) & 255;
          if (at < K) {
            const float2 e = list[(int64_t)i * K + at];
            const int id = __float_as_int(e.y);
            if (id >= 0 && (e.x > bv || (e.x == bv && id < bid))) {
              bv = e.x;
              bid = id;
              bl = 4 * w + q;
            }
          }
        }
      }
    float wv = bv;
    int wid = bid;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const float ov = __shfl_xor_sync(0xffffffffu, wv, o);
      const int oid = __shfl_xor_sync(0xffffffffu, wid, o);
      if (oid != 0x7fffffff && (wid == 0x7fffffff || ov > wv || (ov == wv && oid < wid))) {
        wv = ov;
        wid = oid;
      }
    }
    if (bl >= 0 && bid == wid) {
#pragma unroll
      for (int w = 0; w < 8; ++w)
        if (bl / 4 == w) used[w] += 1u << (8 * (bl % 4));
    }
    if (lane == 0) {
      const bool none = wid == 0x7fffffff;  // only a row of NaN logits has fewer than k
      top_ids[row * k + r] = none ? r : wid;
      top_logprobs[row * k + r] = none ? __uint_as_float(0x7FC00000u) : (wv - m) - logs;
    }
  }
}
constexpr int LP_JOIN_MAX = 1024;  // shares of one row that lp_join_kernel can merge
constexpr int LP_MAX_GROUPS = 128;

// hi, mid and lo of fp32 rows (n, d), ld apart, as three bf16 matrices of row stride ld_o
__global__ void __launch_bounds__(256)
    lp_split_kernel(const float* __restrict__ x, int64_t ld, __nv_bfloat16* __restrict__ out, int64_t ld_o, int64_t rows,
                    int64_t d) {
  pdl_enter();
  const int64_t n = rows * ld_o;
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    const int64_t r = i / ld_o, c = i - r * ld_o;
    const float v = c < d ? x[r * ld + c] : 0.f;
    __nv_bfloat16 hi = __float2bfloat16_rn(v);
    if (isinf(__bfloat162float(hi)) && !isinf(v)) hi = __float2bfloat16_rz(v);
    const float fh = __bfloat162float(hi);
    const float rest = isfinite(v) ? v - fh : 0.f;
    const __nv_bfloat16 mid = __float2bfloat16_rn(rest);
    const __nv_bfloat16 lo = __float2bfloat16_rn(rest - __bfloat162float(mid));
    out[i] = hi;
    out[n + i] = mid;
    out[2 * n + i] = lo;
  }
}

// ---- host side -----------------------------------------------------------------------------------------

LpShape lp_shape(int64_t N, int64_t V, int64_t D, bool f32, int sms) {
  LpShape s;
  s.N = (int)N;
  s.V = (int)V;
  s.kblocks = (int)cdiv(D, 64);
  s.parts = f32 ? 6 : 1;
  s.row_blocks = (int)cdiv(N, 256);
  s.col_tiles = (int)cdiv(V, 256);
  // W's tiles of a group stay in L2 (126 MB, half of it for W) while all rows pass over them
  const int64_t tile_bytes = 256 * (int64_t)s.kblocks * 128 * (f32 ? 3 : 1);
  // (at most 128 groups: a row has then fewer than 2 (148 + 2 * 128) shares)
  const int64_t fit = std::max<int64_t>((64ll << 20) / tile_bytes, cdiv(s.col_tiles, LP_MAX_GROUPS));
  s.group = (int)(fit < s.col_tiles ? fit : s.col_tiles);
  s.total = (int64_t)s.row_blocks * s.col_tiles;
  s.pairs = (int)(s.total < sms / 2 ? s.total : sms / 2);
  const int64_t q = s.total / s.pairs;
  const int64_t most = cdiv(s.group, q) + 1;
  s.slots = (int)(most < s.pairs ? most : s.pairs);
  return s;
}
int lp_groups(const LpShape& s) { return (int)cdiv(s.col_tiles, s.group); }
int lp_list_k(int k) { return k == 0 ? 0 : k <= 8 ? 8 : 32; }

template <int MODE, int K, bool F32>
int lp_launch(const CUtensorMap& th, const CUtensorMap& tw, const CUtensorMap& to, const LpShape& s, const LpArgs& a,
              cudaStream_t st) {
  const int dev = current_device();
  static bool configured[64] = {};
  ULM_REQUIRE(dev >= 0 && dev < 64, "device ordinal %d out of range", dev);
  if (!configured[dev]) {
    ULM_CUDA_TRY(cudaFuncSetAttribute(lp_mma_kernel<MODE, K, F32>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                      (int)LPM_SMEM));
    configured[dev] = true;
  }
  return launch_pdl(lp_mma_kernel<MODE, K, F32>, dim3(2 * s.pairs), dim3(TC_THREADS), LPM_SMEM, st, th, tw, to, s, a);
}

// An operand of the product: bf16 rows, or the three parts of fp32 ones (written to `parts` first).
int lp_operand(CUtensorMap* map, const void* x, int64_t ld, int64_t rows, int64_t D, bool f32, void* parts,
               cudaStream_t st) {
  if (f32) {
    const int64_t ld_o = ulm_operand_ld(D);
    const int64_t ctas = cdiv(rows * ld_o, 256 * 8);
    if (int rc = launch_pdl(lp_split_kernel, dim3((unsigned)(ctas < 8192 ? ctas : 8192)), dim3(256), 0, st,
                            static_cast<const float*>(x), ld, static_cast<__nv_bfloat16*>(parts), ld_o, rows, D))
      return rc;
    return make_tmap(map, Operand{parts, ld_o, rows * ld_o, D, rows, ULM_BF16, false}, 3, 64, 128);
  }
  ULM_REQUIRE(is_aligned16(x) && ld % 8 == 0, "bf16 operands must be 16-byte aligned, their row stride a multiple of 8");
  return make_tmap(map, Operand{x, ld, rows * ld, D, rows, ULM_BF16, false}, 1, 64, 128);
}

}  // namespace
}  // namespace ulm
