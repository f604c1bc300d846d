// The products x = h W^T of the log-probability entries: a tcgen05 kernel on CTA pairs (256 x 256 tiles,
// cta_group::2, operands by TMA, accumulators double-buffered in tensor memory) with three epilogues. The
// logits stay on the SM where no alternatives are asked for; with lists, the chunks of 32 that enter one
// leave it, and LP_DUMP writes them all.
//
// LP_STATS keeps, for each row, the running maximum, sum of exponentials and entropy sum of the softmax in
// registers from tile to tile; an epilogue thread owns half of a row's columns, in chunks of 32 logits.
// The k best logits of a row lie in its k best chunks, by their maxima, so the alternatives take one
// comparison for 32 logits. For many rows an epilogue thread keeps a sorted list of the k best chunks of its
// share and writes a chunk that enters the list to the place of the one that leaves it (about
// k ln(chunks / k) times). LP_DUMP, for few rows, where most chunks of the short shares would enter, writes
// all logits and the maxima of the chunks, and lp_join_kernel picks (2048 x 32000 x 768, k = 20: lists 191
// us, written out 124; 16384 rows: 920 and 1140; no alternatives: 70 and 535, 1500 TFLOP/s).
// LP_GRAD writes the logits' gradient ([v = t] a - p (a + b (log p + H))) for the products that follow: two
// bf16 parts (hi and lo, the output map's batches), or fp32.
//
// Each CTA pair takes one run of consecutive tiles, all of the same length to within one, in an order
// that keeps a row block until its columns are done: h's tile and the rows' state stay, W streams from
// L2. (One column group at a time where W does not fit there.) So all pairs end together whatever N and
// V are, and a row block is cut into at most `slots` shares, which lp_join_kernel adds up,
// looking through the k best chunks of each row.
//
// fp32 operands are given as three bf16 parts each (x = hi + mid + lo to the last bit, lp_split_kernel),
// and the product runs over six pairs of parts, the small ones first: what is left out is up to 2^-24
// of each product (two pairs of a second and a third part). Bound by the tensor cores either way.
#include <algorithm>

#include "gemm.cuh"

namespace ulm {
namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr float LN2 = 0.6931471805599453f;
constexpr int LP_MAX_TOP = 32;  // top_k of the entries

enum { LP_STATS = 0, LP_GRAD = 1, LP_DUMP = 2 };
constexpr int LPM_STAGES = 5;
constexpr int LPM_SLOTS = 2;  // 4 KB staging tiles of an epilogue warp (LP_GRAD)
constexpr uint32_t LPM_HALF_BYTES = 128 * 64 * 2;  // a CTA's 128 rows of one operand, 64 k values
constexpr uint32_t LPM_STAGE_BYTES = 2 * LPM_HALF_BYTES;
constexpr uint32_t LPM_SMEM = LPM_STAGES * LPM_STAGE_BYTES + EPI_WARPS * LPM_SLOTS * 4096u + 1024 + 512;
constexpr int LPM_ROW = 144;  // bytes between the threads' chunks of LP_STATS: no two lanes of a quarter meet
static_assert(32 * LPM_ROW <= LPM_SLOTS * 4096, "a warp's chunks fit its staging tiles");
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
  const int64_t rem = t - r.g * per_group;  // 2^28 rows and more of a wide vocabulary pass 32 bits
  const int wide = min(s.group, s.col_tiles - r.g * s.group);
  r.rb = (int)(rem / wide);
  r.ct = r.g * s.group + (int)(rem - (int64_t)r.rb * wide);
  return r;
}

// What an epilogue reads and writes.
struct LpArgs {
  const int64_t* tokens;
  // LP_STATS: for share i = ((row * groups + g) * slots + slot) * 2 + half of a row: (max, sum, entropy sum)
  // in part[4 i] (base 2: of 2^(x log2 e - max log2 e)); its k best chunks in list[i * k + j], descending, as
  // (maximum, chunk index * 32 + place), their logits in dump[(i * k + place) * 32]; and given[row], the
  // token's logit
  float* part;
  float2* list;
  float* dump;
  float* given;
  int k;
  // LP_DUMP: besides part and given, the largest logit of each chunk of 32 columns in
  // chunk_max[row * ld_max + column / 32] (the logits themselves go through the output's tensor map)
  float* chunk_max;
  int64_t ld_max;
  int groups;
  // LP_GRAD
  const float* stats;
  const float* entropy;
  const float* dlogprobs;
  const float* dentropy;
};

// The backward's factors of one row: dx_v = [v = t] a - p_v (a + b (log p_v + H)), with p_v = 2^l,
// l = (x_v - m) log2 e - l2, b2 = b ln 2.
struct LpCoef {
  float m, l2, c0, b2, a;
  int64_t t;
  // the second term. A masked logit (l = -inf) has p = 0: l is kept at -200, whose power is 0 too. A row of
  // NaN statistics has a NaN c0.
  __device__ __forceinline__ float others(float x) const {
    const float l = fmaxf(fmaf(x - m, LOG2E, -l2), -200.f);
    return -fast_exp2(l) * fmaf(b2, l, c0);
  }
  __device__ __forceinline__ void others2(float& x, float& y) const {
    float lx, ly;
    f32x2_split(f32x2_fma(f32x2_add(f32x2(x, y), f32x2(-m, -m)), f32x2(LOG2E, LOG2E), f32x2(-l2, -l2)), lx, ly);
    lx = fmaxf(lx, -200.f);
    ly = fmaxf(ly, -200.f);
    const uint64_t q = f32x2_fma(f32x2(-b2, -b2), f32x2(lx, ly), f32x2(-c0, -c0));
    f32x2_split(f32x2_mul(f32x2(fast_exp2(lx), fast_exp2(ly)), q), x, y);
  }
};
__device__ __forceinline__ LpCoef lp_coef(const int64_t* tokens, const float* stats, const float* entropy,
                                          const float* dlogprobs, const float* dentropy, int64_t r, int V) {
  LpCoef c;
  c.t = tokens[r];
  c.m = stats[2 * r];
  c.l2 = stats[2 * r + 1] * LOG2E;
  c.a = c.t == -1 || !dlogprobs ? 0.f : dlogprobs[r];
  if (dlogprobs && (c.t < -1 || c.t >= V)) c.a = __uint_as_float(0x7FC00000u);  // (the entropy does not see t)
  const float b = dentropy ? dentropy[r] : 0.f;
  c.b2 = b * LN2;
  c.c0 = c.a + (b != 0.f ? b * entropy[r] : 0.f);
  if (!(c.l2 < INFINITY && c.l2 > -INFINITY)) c.c0 = __uint_as_float(0x7FC00000u);
  return c;
}

// The statistics of one thread's share of a row, over chunks of 32 logits; K is the most chunks that its
// list can hold, the first K - k places are taken by +inf.
template <int K>
struct LpRun {
  float m, m2, s, u;  // maximum (at least -1e30), m log2 e, sum 2^(x log2 e - m2), sum 2^(.) (.)
  float last;         // maximum of the chunk added last
  float v[K > 0 ? K : 1];
  int id[K > 0 ? K : 1];

  __device__ __forceinline__ void reset(bool live, int k) {
    m = -1e30f;
    m2 = __fmul_rn(m, LOG2E);
    s = u = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      v[j] = live && j >= K - k ? -INFINITY : INFINITY;  // nothing enters the list of a row that is not there
      id[j] = -32 + (j - (K - k));
    }
  }
  // logits x of columns col0 .. col0 + 31, V the first column past the last; dump: this share's chunks in
  // global memory, stage: this thread's 128 bytes of shared memory. A chunk that enters the list leaves by a
  // bulk copy of its own: 32 rows' chunks lie far apart, and plain stores of them kept the warp waiting.
  __device__ __forceinline__ void add(float (&x)[32], int col0, int V, float* dump, uint8_t* stage) {
    if (col0 + 32 > V) {
#pragma unroll
      for (int i = 0; i < 32; ++i) x[i] = col0 + i < V ? x[i] : -1e35f;  // no power, in any row
    }
    float lm = fmaxf(x[0], x[1]);
#pragma unroll
    for (int i = 2; i < 32; i += 2) lm = fmaxf(lm, fmaxf(x[i], x[i + 1]));
    last = lm;
    if (K > 0) {
      if (lm > v[K - 1]) {
        const int place = id[K - 1] & 31, mine = col0 | place;
#pragma unroll
        for (int j = K - 1; j > 0; --j) {
          const bool up = lm > v[j - 1], here = lm > v[j];
          v[j] = up ? v[j - 1] : here ? lm : v[j];
          id[j] = up ? id[j - 1] : here ? mine : id[j];
        }
        if (lm > v[0]) {
          v[0] = lm;
          id[0] = mine;
        }
        // the chunk before has left the stage and has landed: it may be the one whose place is taken now, and
        // two copies in flight to one address have no order
        bulk_wait_group<0>();
        float4* d = reinterpret_cast<float4*>(stage);
#pragma unroll
        for (int i = 0; i < 8; ++i) d[i] = make_float4(x[4 * i], x[4 * i + 1], x[4 * i + 2], x[4 * i + 3]);
        fence_proxy_async_smem();
        bulk_store(dump + place * 32, stage, 128);
        bulk_commit_group();
      }
      __syncwarp();
    }
    if (lm > m) {
      const float n2 = __fmul_rn(lm, LOG2E), d = m2 - n2, f = fast_exp2(d);
      u = f > 0.f ? (u + s * d) * f : 0.f;
      s *= f;
      m = lm;
      m2 = n2;
    }
    const uint64_t scale = f32x2(LOG2E, LOG2E), shift = f32x2(-m2, -m2);
    uint64_t ss[2] = {0, 0}, uu[2] = {0, 0};
#pragma unroll
    for (int i = 0; i < 32; i += 2) {
      const uint64_t d = f32x2_fma(f32x2(x[i], x[i + 1]), scale, shift);
      float d0, d1;
      f32x2_split(d, d0, d1);
      const uint64_t e = f32x2(fast_exp2(d0), fast_exp2(d1));
      ss[i / 2 % 2] = f32x2_add(ss[i / 2 % 2], e);
      uu[i / 2 % 2] = f32x2_fma(e, d, uu[i / 2 % 2]);
    }
    float s0, s1, u0, u1;
    f32x2_split(f32x2_add(ss[0], ss[1]), s0, s1);
    f32x2_split(f32x2_add(uu[0], uu[1]), u0, u1);
    s += s0 + s1;
    u += u0 + u1;
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
    if (MODE != LP_STATS) tma_prefetch_desc(&tma_out);
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
    float* dump = nullptr;  // the chunks of this thread's share
    int64_t share = 0;
    if (MODE != LP_GRAD) run.reset(false, 0);
    auto flush = [&]() {
      if (MODE == LP_GRAD || at_rb < 0 || !live) return;
      *reinterpret_cast<float4*>(args.part + 4 * share) = make_float4(run.m, run.s, run.u, 0.f);
      if (K > 0) {
#pragma unroll
        for (int q = 0; q < K; ++q)
          if (q >= K - args.k) args.list[share * args.k + q - (K - args.k)] = make_float2(run.v[q], __int_as_float(run.id[q]));
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
        if (MODE != LP_GRAD) {
          const int slot = pair - lp_pair_of(shape, lp_row_first(shape, at_g, at_rb));
          share = ((row * args.groups + at_g) * shape.slots + slot) * 2 + half;
          dump = args.dump + share * args.k * 32;
          run.reset(live, args.k);
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
      if (MODE != LP_GRAD) {
        uint32_t ra[32], rb[32];
        float4 cmax = make_float4(0.f, 0.f, 0.f, 0.f);
        // a list of 32 leaves no registers for the next chunk's load ahead
        constexpr bool AHEAD = K <= 8;
        if (AHEAD && chunks > 0) tmem_ld_32x32_issue(taddr, ra);
        auto one = [&](uint32_t (&r)[32], uint32_t (&next)[32], int ch) {
          const int col0 = col_base + 32 * ch;
          if (!AHEAD) tmem_ld_32x32_issue(taddr + 32 * ch, r);
          tmem_ld_32x32_wait(r);
          if (AHEAD && ch + 1 < chunks) tmem_ld_32x32_issue(taddr + 32 * (ch + 1), next);
          float x[32];
#pragma unroll
          for (int i = 0; i < 32; ++i) x[i] = __uint_as_float(r[i]);
          run.add(x, col0, shape.V, dump, slots + lane * LPM_ROW);
          if (tok >= col0 && tok < col0 + 32 && tok < shape.V) {
            float g = 0.f;
#pragma unroll
            for (int i = 0; i < 32; ++i)
              if (col0 + i == (int)tok) g = x[i];
            args.given[row] = g;
          }
          if (MODE == LP_DUMP) {
            (ch == 0 ? cmax.x : ch == 1 ? cmax.y : ch == 2 ? cmax.z : cmax.w) = run.last;
            uint8_t* out = slots + (n % LPM_SLOTS) * 4096;
            ++n;
            if (lane == 0) bulk_wait_group_read<LPM_SLOTS - 1>();  // the store before last has read its slot
            __syncwarp();
            stage_write<true, 32>(out, lane, 0, x);
            fence_proxy_async_smem();
            __syncwarp();
            if (lane == 0) {
              tma_store_3d(&tma_out, out, col0, tile.rb * 256 + (int)rank * 128 + quad * 32, 0);
              bulk_commit_group();
            }
          }
          __syncwarp();
        };
        if (AHEAD) {
#pragma unroll
          for (int ch = 0; ch < 4; ch += 2) {
            if (ch < chunks) one(ra, rb, ch);
            if (ch + 1 < chunks) one(rb, ra, ch + 1);
          }
        } else {
#pragma unroll 1
          for (int ch = 0; ch < chunks; ++ch) one(ra, rb, ch);
        }
        if (MODE == LP_DUMP && live && chunks > 0)  // rows of chunk_max are whole tiles long
          *reinterpret_cast<float4*>(args.chunk_max + row * args.ld_max + col_base / 32) = cmax;
      } else {
        constexpr int CW = F32 ? 32 : 64;  // columns of a staged chunk of 128 bytes a row
        const int nch = rows_here ? min(128 / CW, (shape.V - col_base + CW - 1) / CW) : 0;
#pragma unroll 1
        for (int i = 0; i < nch; ++i) {
          uint8_t* out = slots + (n % LPM_SLOTS) * 4096;
          ++n;
          if (lane == 0) {
            if (!F32)
              bulk_wait_group_read<0>();  // the two parts take both slots
            else
              bulk_wait_group_read<LPM_SLOTS - 1>();  // the store before last has read its slot
          }
          __syncwarp();
#pragma unroll
          for (int hh = 0; hh < CW / 32; ++hh) {
            float v[32];
            const int col0 = col_base + i * CW + hh * 32;
            tmem_ld_32x32(taddr + (uint32_t)(i * CW + hh * 32), v);
#pragma unroll
            for (int q = 0; q < 32; q += 2) c.others2(v[q], v[q + 1]);
            if (tok >= col0 && tok < col0 + 32) {
#pragma unroll
              for (int q = 0; q < 32; ++q)
                if (col0 + q == (int)tok) v[q] += c.a;
            }
            __syncwarp();
            stage_write<F32, 32>(out, lane, hh * (F32 ? 8 : 4), v);
            if (!F32) {
#pragma unroll
              for (int q = 0; q < 32; ++q) v[q] -= __bfloat162float(__float2bfloat16_rn(v[q]));
              stage_write<F32, 32>(slots + (n % LPM_SLOTS) * 4096, lane, hh * 4, v);
            }
          }
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            const int r0 = tile.rb * 256 + (int)rank * 128 + quad * 32;
            tma_store_3d(&tma_out, out, col_base + i * CW, r0, 0);
            if (!F32) tma_store_3d(&tma_out, slots + (n % LPM_SLOTS) * 4096, col_base + i * CW, r0, 1);
            bulk_commit_group();
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive_cluster_relaxed(leader_tempty + (uint32_t)(acc * sizeof(uint64_t)));
    }
    flush();
    bulk_wait_group<0>();
  }

  tc_fence_before();
  cluster_sync_all();  // all MMAs done and all TMEM reads finished in both CTAs
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem_base, 512);
  }
}

// Order of the alternatives as one integer: the value's bits made monotone (NaN above all, -0 = 0),
// then the lower id.
__device__ __forceinline__ uint64_t lp_key(float x, uint32_t id) {
  uint32_t b = __float_as_uint(x + 0.f);
  b = (b & 0x80000000u) ? ~b : (b | 0x80000000u);
  if (x != x) b = 0xFFFFFFFEu;
  return ((uint64_t)b << 32) | (uint64_t)(0xFFFFFFFFu - id);
}
__device__ __forceinline__ float lp_key_value(uint64_t k) {
  const uint32_t b = (uint32_t)(k >> 32);
  if (b == 0xFFFFFFFEu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((b & 0x80000000u) ? (b & 0x7FFFFFFFu) : ~b);
}
__device__ __forceinline__ uint32_t lp_key_id(uint64_t k) { return 0xFFFFFFFFu - (uint32_t)k; }

// TPR threads per row (a warp for many rows, 128 threads for few): the shares' statistics merged, then
// the k best logits of the row's chunks. Of the shares' lists only those with the k best first chunks can
// hold one of the row's k best chunks, and of the row's logits only those in its k best chunks (a chunk
// with k better ones ahead of it, in the order of maximum and column, has k better logits ahead of all of
// its own). Each of the three choices is a rank among at most 1024 keys, about k of them in the last two.
// DUMP: the logits are there whole, with the maximum of each chunk: the best chunks are looked for among
// those not under the k-th largest of 64 groups' maxima.
constexpr int LP_JOIN_MAX = 1024;  // shares of one row, and chunks or logits to choose from
constexpr int LP_JOIN_GROUPS = 64;
constexpr int LP_JOIN_ROWS = 2;    // rows of a CTA when a warp has a row
template <int TPR, bool DUMP>
__global__ void __launch_bounds__(TPR == 32 ? 32 * LP_JOIN_ROWS : TPR)
    lp_join_kernel(const LpShape shape, const LpArgs args, float* __restrict__ logprobs, float* __restrict__ entropy,
                   float* __restrict__ stats, int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs,
                   int room) {
  constexpr int ROWS = TPR == 32 ? LP_JOIN_ROWS : 1;
  extern __shared__ uint64_t join_smem[];  // of each row: `room` keys, and as many places
  __shared__ int chosen[ROWS][LP_MAX_TOP];
  __shared__ uint64_t best_key[ROWS][LP_MAX_TOP];
  __shared__ int counts[ROWS][3];
  __shared__ uint64_t bound[ROWS];
  __shared__ float4 wred[TPR / 32];
  __shared__ float gmax[DUMP ? TPR : 1];
  __shared__ float thr_s;
  pdl_enter();
  const int tid = threadIdx.x % TPR, w = threadIdx.x / TPR;
  const int64_t row = (int64_t)blockIdx.x * ROWS + w;
  if (row >= shape.N) return;
  uint64_t* key = join_smem + w * room;
  int* at = reinterpret_cast<int*>(join_smem + ROWS * room) + w * room;
  auto sync = [] {
    if (TPR == 32)
      __syncwarp();
    else
      __syncthreads();
  };
  const int rb = (int)(row / 256), k = args.k;
  const int all = args.groups * shape.slots * 2;  // the row's possible shares
  // whether share i is there: its pair took tiles of this row block
  auto slots_of = [&](int g) {
    const int64_t a = lp_row_first(shape, g, rb), b = a + min(shape.group, shape.col_tiles - g * shape.group);
    return lp_pair_of(shape, b - 1) - lp_pair_of(shape, a) + 1;
  };
  const int slots0 = slots_of(0);
  auto there = [&](int i) {
    const int g = args.groups == 1 ? 0 : i / (2 * shape.slots);
    return i < all && i / 2 - g * shape.slots < (g == 0 ? slots0 : slots_of(g));
  };
  if (tid < 3) counts[w][tid] = 0;
  const float4* part = reinterpret_cast<const float4*>(args.part) + row * all;
  const float2* list = args.list + row * all * k;
  const float* dump = args.dump + row * all * k * 32;
  // sums are relative to m2 = fl(max log2 e), here as in the shares
  float m = -1e30f, m2 = __fmul_rn(m, LOG2E), s = 0.f, u = 0.f;
  auto merge = [&](float om, float os, float ou) {
    const float M = fmaxf(m, om), M2 = __fmul_rn(M, LOG2E);
    const float da = m2 - M2, fa = fast_exp2(da), db = __fmul_rn(om, LOG2E) - M2, fb = fast_exp2(db);
    u = (fa > 0.f ? (u + s * da) * fa : 0.f) + (fb > 0.f ? (ou + os * db) * fb : 0.f);
    s = s * fa + os * fb;
    m = M;
    m2 = M2;
  };
  sync();
  for (int i = tid; i < all; i += TPR) {
    if (!there(i)) continue;
    const float4 p = part[i];
    if (!DUMP && k > 0) {  // the share's first chunk
      const float2 e = list[(int64_t)i * k];
      const int id = __float_as_int(e.y);
      if (id >= 0) {
        const int to = atomicAdd(&counts[w][0], 1);
        key[to] = lp_key(e.x, (uint32_t)(id >> 5));
        at[to] = i;
      }
    }
    merge(p.x, p.y, p.z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const float om = __shfl_xor_sync(0xffffffffu, m, o), os = __shfl_xor_sync(0xffffffffu, s, o),
                ou = __shfl_xor_sync(0xffffffffu, u, o);
    merge(om, os, ou);
  }
  if (TPR > 32) {
    if ((tid & 31) == 0) wred[tid >> 5] = make_float4(m, s, u, 0.f);
    sync();
    m = -1e30f;
    m2 = __fmul_rn(m, LOG2E);
    s = u = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) merge(wred[i].x, wred[i].y, wred[i].z);
  }
  // logp = (x - m) - logs: log s, and how far m2 is from m log2 e. No power is left of a row below -1e30
  // throughout, or past 2.3e38: NaN.
  const float logs = s > 0.f ? logf(s) + fmaf(-m, LOG2E, m2) * LN2 : __uint_as_float(0x7FC00000u);
  if (tid == 0) {
    const int64_t t = args.tokens[row];
    logprobs[row] = t == -1 ? 0.f : t < 0 || t >= shape.V ? __uint_as_float(0x7FC00000u) : (args.given[row] - m) - logs;
    entropy[row] = logf(s) - LN2 * (u / s);
    if (stats) {
      stats[2 * row] = m;
      stats[2 * row + 1] = logs;
    }
  }
  if (k == 0) return;
  // f(key index, rank) for the keys among the k best of n (all different)
  auto rank = [&](int n, auto&& f) {
    for (int c = tid; c < n; c += TPR) {
      const uint64_t mine = key[c];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < n; ++j) r += key[j] > mine ? 1 : 0;
      if (r < k) f(c, r);
    }
  };
  int best = 0;
  if (!DUMP) {
    sync();
    const int heads = counts[w][0], lists = min(heads, k);
    rank(heads, [&](int c, int r) {
      chosen[w][r] = at[c];
      if (r == k - 1) bound[w] = key[c];
    });
    sync();
    const uint64_t floor_key = heads >= k ? bound[w] : 0;  // the k-th best first chunk
    // the chosen lists' chunks that are not under it
#pragma unroll 4
    for (int i = tid; i < lists * 32; i += TPR) {
      const int l = chosen[w][i / 32], j = i % 32;
      if (j >= k) continue;
      const float2 e = list[(int64_t)l * k + j];
      const int id = __float_as_int(e.y);
      const uint64_t kk = lp_key(e.x, (uint32_t)(id >> 5));
      if (id >= 0 && kk >= floor_key) {
        const int to = atomicAdd(&counts[w][1], 1);
        key[to] = kk;
        at[to] = l * k + (id & 31);
      }
    }
    sync();
    const int chunks = counts[w][1];
    best = min(chunks, k);
    rank(chunks, [&](int c, int r) { chosen[w][r] = c; });
    sync();
  } else {
    const int chunks = (shape.V + 31) / 32;
    const float* cm = args.chunk_max + row * args.ld_max;
    best = min(chunks, k);
    float g = -INFINITY;
#pragma unroll 4
    for (int i = tid; i < chunks; i += TPR) g = fmaxf(g, cm[i]);
    gmax[tid] = g;
    if (tid == 0) thr_s = -INFINITY;
    sync();
    if (tid < LP_JOIN_GROUPS) {
      float mine = gmax[tid];
#pragma unroll
      for (int j = 1; j < TPR / LP_JOIN_GROUPS; ++j) mine = fmaxf(mine, gmax[tid + j * LP_JOIN_GROUPS]);
      gmax[tid] = mine;
    }
    sync();
    if (tid < LP_JOIN_GROUPS) {
      const float mine = gmax[tid];
      int r = 0;
#pragma unroll 8
      for (int j = 0; j < LP_JOIN_GROUPS; ++j) r += (gmax[j] > mine || (gmax[j] == mine && j < tid)) ? 1 : 0;
      if (r == k - 1) thr_s = mine;
    }
    sync();
    const float thr = thr_s;
#pragma unroll 4
    for (int i = tid; i < chunks; i += TPR) {
      const float x = cm[i];
      if (x >= thr) {
        const int to = atomicAdd(&counts[w][1], 1);
        if (to < room) {
          key[to] = lp_key(x, (uint32_t)i);
          at[to] = i;
        }
      }
    }
    sync();
    const int n = counts[w][1];
    if (n <= room) {
      best = min(n, k);  // fewer only where a chunk is all NaN
      rank(n, [&](int c, int r) { chosen[w][r] = c; });
      sync();
    } else {
      // many equal maxima: the best one after the last, k times
      uint64_t last = ~0ull;
      for (int j = 0; j < best; ++j) {
        uint64_t top = 0;
        for (int i = tid; i < chunks; i += TPR) {
          const uint64_t kk = lp_key(cm[i], (uint32_t)i);
          if (kk < last && kk > top) top = kk;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
          const uint64_t other = __shfl_xor_sync(0xffffffffu, top, o);
          top = other > top ? other : top;
        }
        sync();
        if ((tid & 31) == 0) best_key[w][tid >> 5] = top;
        sync();
#pragma unroll
        for (int i = 0; i < TPR / 32; ++i) top = best_key[w][i] > top ? best_key[w][i] : top;
        last = top;
        if (tid == 0) {
          key[j] = top;
          at[j] = (int)lp_key_id(top);
          chosen[w][j] = j;
        }
      }
      sync();
    }
  }
  // the best chunks; the last one's maximum bounds the k-th best logit from below
  int mine_at = 0;
  if (tid < best) {
    best_key[w][tid] = key[chosen[w][tid]];
    mine_at = at[chosen[w][tid]];
  }
  sync();
  if (tid < best) chosen[w][tid] = mine_at;
  sync();
  const float least = best == k ? lp_key_value(best_key[w][k - 1]) : -INFINITY;
#pragma unroll 4
  for (int i = tid; i < best * 32; i += TPR) {
    const uint32_t id = lp_key_id(best_key[w][i / 32]) * 32 + i % 32;
    const float x = DUMP ? (id < (uint32_t)shape.V ? args.dump[row * args.ld_max * 32 + id] : -INFINITY)
                         : dump[(int64_t)chosen[w][i / 32] * 32 + i % 32];
    if (id < (uint32_t)shape.V && x >= least) key[atomicAdd(&counts[w][2], 1)] = lp_key(x, id);
  }
  sync();
  const int n = counts[w][2];
  rank(n, [&](int c, int r) {
    top_ids[row * k + r] = lp_key_id(key[c]);
    top_logprobs[row * k + r] = (lp_key_value(key[c]) - m) - logs;
  });
  // Only a row with NaN or -inf among its logits has fewer than k others: the lowest ids that are not there yet
  // (of the first k at least k - n are free) take the places left.
  if (n < k && tid < k) {
    auto taken = [&](uint32_t id) {
      for (int j = 0; j < n; ++j)
        if (lp_key_id(key[j]) == id) return true;
      return false;
    };
    int place = n;
    for (int c = 0; c < tid; ++c) place += taken((uint32_t)c) ? 0 : 1;
    if (place < k && !taken((uint32_t)tid)) {
      top_ids[row * k + place] = tid;
      top_logprobs[row * k + place] = __uint_as_float(0x7FC00000u);
    }
  }
}
constexpr int LP_MAX_GROUPS = 128;

// hi, mid and lo of fp32 rows (n, d), ld apart, as three bf16 matrices of row stride ld_o (a multiple of 8,
// the rest zero); a thread takes two neighbours
__global__ void __launch_bounds__(256)
    lp_split_kernel(const float* __restrict__ x, int64_t ld, __nv_bfloat16* __restrict__ out, int64_t ld_o, int64_t rows,
                    int64_t d) {
  pdl_enter();
  const int64_t part = rows * ld_o / 2;  // pairs of one matrix
  uint32_t* o = reinterpret_cast<uint32_t*>(out);
  auto split = [](float v, __nv_bfloat16& hi, __nv_bfloat16& mid, __nv_bfloat16& lo) {
    hi = __float2bfloat16_rn(v);
    if (isinf(__bfloat162float(hi)) && !isinf(v)) hi = __float2bfloat16_rz(v);
    const float rest = isfinite(v) ? v - __bfloat162float(hi) : 0.f;
    mid = __float2bfloat16_rn(rest);
    lo = __float2bfloat16_rn(rest - __bfloat162float(mid));
  };
  for (int64_t r = blockIdx.x; r < rows; r += gridDim.x) {
    const float* row = x + r * ld;
#pragma unroll 4
    for (int64_t c = threadIdx.x; c < ld_o / 2; c += 256) {
      __nv_bfloat162 p[3];
      split(2 * c < d ? row[2 * c] : 0.f, p[0].x, p[1].x, p[2].x);
      split(2 * c + 1 < d ? row[2 * c + 1] : 0.f, p[0].y, p[1].y, p[2].y);
#pragma unroll
      for (int i = 0; i < 3; ++i) o[i * part + r * (ld_o / 2) + c] = *reinterpret_cast<const uint32_t*>(&p[i]);
    }
  }
}

int lp_split(const float* x, int64_t ld, void* out, int64_t ld_o, int64_t rows, int64_t d, cudaStream_t st) {
  return launch_pdl(lp_split_kernel, dim3((unsigned)std::min<int64_t>(rows, 1 << 20)), dim3(256), 0, st, x, ld,
                    static_cast<__nv_bfloat16*>(out), ld_o, rows, d);
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
// Keys of one row of lp_join_kernel: the first chunks of its shares, chunks of k lists, logits of k chunks.
int lp_join_room(int shares, int k) { return std::max(shares, 32 * k); }
int lp_groups(const LpShape& s) { return (int)cdiv(s.col_tiles, s.group); }
constexpr int LP_LIST = 8, LP_LONG_LIST = 32;  // chunks in a register list

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
    if (int rc = lp_split(static_cast<const float*>(x), ld, parts, ld_o, rows, D, st)) return rc;
    return make_tmap(map, Operand{parts, ld_o, rows * ld_o, D, rows, ULM_BF16, false}, 3, 64, 128);
  }
  ULM_REQUIRE(is_aligned16(x) && ld % 8 == 0, "bf16 operands must be 16-byte aligned, their row stride a multiple of 8");
  return make_tmap(map, Operand{x, ld, rows * ld, D, rows, ULM_BF16, false}, 1, 64, 128);
}

}  // namespace
}  // namespace ulm
