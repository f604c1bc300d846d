// Log probabilities of given tokens, with the distribution's entropy and its best alternatives:
//   m = max_v x_v, s = sum_v exp(x_v - m), u = sum_v exp(x_v - m) (x_v - m)
//   logp_t = (x_t - m) - log s,   H = log s - u / s,   top k by (value descending, id ascending)
// and backward, from the gradients a of logp_t and b of H:
//   dx_v = a ([v = t] - p_v) - b p_v (log p_v + H),   p_v = exp((x_v - m) - log s)
// over rows of logits x that exist already (ulm_token_logprobs_*), or that are x = h W^T
// (ulm_lm_head_logprobs_*). Token -1 is padding: logp 0 and no a term. Any other token outside
// [0, V) makes its row's logp and gradients NaN. All statistics are fp32.
#include "logprobs_mma.cu"

namespace ulm {
namespace {

constexpr int LP_THREADS = 256;
constexpr int LP_GROUPS = 64;     // groups of threads whose maxima give the threshold of the top k
constexpr int LP_CAP = 512;       // candidates of one CTA above the threshold
constexpr int LP_MAX_SPLIT = 8;   // CTAs (one cluster) that share a row

// Running statistics of a set of logits in base 2: the maximum m (at least -1e30), m2 = fl(m log2 e),
// s = sum 2^(x log2 e - m2) and u = sum 2^(.) (.).
struct LpStat {
  float m, m2, s, u;
  __device__ __forceinline__ void raise(float to) {
    const float n2 = __fmul_rn(to, LOG2E), d = m2 - n2, f = fast_exp2(d);
    u = f > 0.f ? (u + s * d) * f : 0.f;
    s *= f;
    m = to;
    m2 = n2;
  }
};
constexpr float LP_LEAST = -1e30f;

__device__ __forceinline__ LpStat lp_merge(LpStat a, LpStat b) {
  const float M = fmaxf(a.m, b.m);
  a.raise(M);
  b.raise(M);
  a.s += b.s;
  a.u += b.u;
  return a;
}

// NV more logits into a thread's statistics: the largest and the smallest first. Logits below -1e30 (-inf,
// or the type's lowest value, is a mask) count as -1e35, whose power is 0 too, but whose product with it is
// no 0 times -inf.
// Returns the largest, or +inf once the sum is NaN.
template <int NV>
__device__ __forceinline__ float lp_add(LpStat& st, const float (&given)[NV]) {
  float x[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) x[i] = given[i];
  float hi = x[0], lo = x[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) {
    hi = fmaxf(hi, x[i]);
    lo = fminf(lo, x[i]);
  }
  if (hi > st.m) st.raise(hi);
  if (lo < LP_LEAST) {
#pragma unroll
    for (int i = 0; i < NV; ++i) x[i] = x[i] < LP_LEAST ? -1e35f : x[i];
  }
  float s1 = 0.f, u1 = 0.f;
  if (NV % 2 == 0) {
    const uint64_t scale = f32x2(LOG2E, LOG2E), shift = f32x2(-st.m2, -st.m2);
    uint64_t ss = 0, uu = 0;
#pragma unroll
    for (int i = 0; i + 1 < NV; i += 2) {
      const uint64_t d = f32x2_fma(f32x2(x[i], x[i + 1]), scale, shift);
      float d0, d1;
      f32x2_split(d, d0, d1);
      const uint64_t e = f32x2(fast_exp2(d0), fast_exp2(d1));
      ss = f32x2_add(ss, e);
      uu = f32x2_fma(e, d, uu);
    }
    float s2, u2;
    f32x2_split(ss, s1, s2);
    f32x2_split(uu, u1, u2);
    s1 += s2;
    u1 += u2;
  } else {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      const float d = fmaf(x[i], LOG2E, -st.m2), e = fast_exp2(d);
      s1 += e;
      u1 = fmaf(e, d, u1);
    }
  }
  st.s += s1;
  st.u += u1;
  return st.s == st.s ? hi : INFINITY;
}

template <typename T>
__device__ __forceinline__ float lp_load(const T* p);
template <>
__device__ __forceinline__ float lp_load<float>(const float* p) {
  return *p;
}
template <>
__device__ __forceinline__ float lp_load<__nv_bfloat16>(const __nv_bfloat16* p) {
  return __bfloat162float(*p);
}

// Logits of 16 bytes as floats, and back.
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float* x) {
    x[0] = __uint_as_float(q.x);
    x[1] = __uint_as_float(q.y);
    x[2] = __uint_as_float(q.z);
    x[3] = __uint_as_float(q.w);
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    return make_uint4(__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]));
  }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float* x) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
  static __device__ __forceinline__ uint4 pack(const float* x) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const __nv_bfloat162 h = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
      w[i] = *reinterpret_cast<const uint32_t*>(&h);
    }
    return make_uint4(w[0], w[1], w[2], w[3]);
  }
};

// Pieces of a thread in flight: 16 values.
template <typename T>
constexpr int LP_UNROLL = 16 / LpVec<T>::N;
// CTAs an SM, by the registers that the batches leave (8192 x 32000 bf16: 6 CTAs 99 us, 5 106; fp32 is
// faster with 5)
template <typename T>
constexpr int LP_CTAS = LpVec<T>::N == 8 ? 6 : 5;
constexpr int LP_KEPT = 16;  // batches of a thread whose maxima are kept for the second look

// Elements before the first 16-byte boundary at p, at most n.
template <typename T>
__device__ __forceinline__ int lp_head(const T* p, int n) {
  const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15) / sizeof(T));
  return h < n ? h : n;
}

// f(batch, ids, values) over logits c0 .. c1 of a row, from its first 16-byte boundary in batches of U 16-byte
// pieces a thread (batch 0, 1, ... of the thread), loaded while the ones before are used; batch -1 for the
// pieces and, at the two ends, the logits that are left. AGAIN: a later look, at the batches that
// want(batch) names and at what is left.
template <typename T, int U, bool AGAIN, typename W, typename F>
__device__ __forceinline__ void lp_for_each(const T* row, int c0, int c1, W&& want, F&& f) {
  constexpr int NV = LpVec<T>::N;
  const int n = c1 - c0, head = lp_head(row + c0, n), nvec = (n - head) / NV, tail0 = c0 + head + nvec * NV;
  const uint4* body = reinterpret_cast<const uint4*>(row + c0 + head);
  auto one = [&](int id) {
    const float x[1] = {lp_load(row + id)};
    const int ids[1] = {id};
    f(-1, ids, x);
  };
  if ((int)threadIdx.x < head) one(c0 + (int)threadIdx.x);
  uint4 ahead[U];
  auto load = [&](int i) {
#pragma unroll
    for (int j = 0; j < U; ++j)
      if (i + j * LP_THREADS < nvec) ahead[j] = body[i + j * LP_THREADS];
  };
  if (!AGAIN) load(threadIdx.x);
  int batch = 0;
  for (int i = threadIdx.x; i < nvec; i += U * LP_THREADS, ++batch) {
    const bool whole = i + (U - 1) * LP_THREADS < nvec;
    if (AGAIN) {
      if (whole && !want(batch)) continue;
      load(i);
    }
    uint4 q[U];
#pragma unroll
    for (int j = 0; j < U; ++j) q[j] = ahead[j];
    if (!AGAIN) load(i + U * LP_THREADS);
    if (whole) {
      float x[U * NV];
      int ids[U];
#pragma unroll
      for (int j = 0; j < U; ++j) {
        LpVec<T>::unpack(q[j], x + j * NV);
        ids[j] = c0 + head + (i + j * LP_THREADS) * NV;
      }
      f(batch, ids, x);
    } else {
#pragma unroll
      for (int j = 0; j < U - 1; ++j) {
        if (i + j * LP_THREADS >= nvec) break;
        float x[NV];
        LpVec<T>::unpack(q[j], x);
        const int ids[1] = {c0 + head + (i + j * LP_THREADS) * NV};
        f(-1, ids, x);
      }
    }
  }
  if (tail0 + (int)threadIdx.x < c1) one(tail0 + (int)threadIdx.x);
}

// The row's logp of its token from its statistics.
template <typename T>
__device__ __forceinline__ float lp_given(const T* row, int64_t t, int V, float base, float logs) {
  if (t == -1) return 0.f;
  if (t < 0 || t >= V) return __uint_as_float(0x7FC00000u);
  return (lp_load(row + t) - base) - logs;
}

__device__ __forceinline__ uint64_t lp_block_max(uint64_t v, uint64_t* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t other = __shfl_xor_sync(0xffffffffu, v, o);
    v = other > v ? other : v;
  }
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  v = red[0];
#pragma unroll
  for (int w = 1; w < LP_THREADS / 32; ++w) v = red[w] > v ? red[w] : v;
  return v;
}

// One cluster of `split` CTAs per row, each with an equal run of its columns. A CTA makes one pass over
// its logits for the statistics and, for the alternatives, a second look at those batches whose maximum
// reaches a threshold: the k-th largest of 64 groups' maxima bounds the k-th best logit of the run from
// below, and only about k logits reach it. The cluster's first CTA joins the runs. Bound by arithmetic for many
// rows (4096 x 32000 bf16: 57 us, 4.6 TB/s, DRAM at 57%; the powers' pipe is at 64%, the issue slots at 71%),
// by latency for few: a row of 32000 fp32 split over 8 CTAs takes 3.8 us without alternatives and 6.1 with 5.
// Where a mask leaves fewer than k logits, the k passes of the second form show: 256 rows of 32000 fp32 with
// three open tokens take 18 us for k = 1 and 156 for k = 20, 4096 rows 111 and 1916 (125 with all open).
template <typename T>
__global__ void __launch_bounds__(LP_THREADS, LP_CTAS<T>)
    lp_rows_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens,
                   float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ stats,
                   int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs, int V, int k, int split) {
  __shared__ float wmax[LP_THREADS / 32];
  __shared__ float2 wsum[LP_THREADS / 32];
  __shared__ alignas(16) LpStat runs[LP_MAX_SPLIT];                    // of the cluster's CTAs (first CTA)
  __shared__ uint64_t best[LP_MAX_SPLIT * LP_MAX_TOP];     // their alternatives (first CTA)
  __shared__ alignas(16) float gmax[LP_GROUPS];
  __shared__ float kept[LP_KEPT * LP_THREADS];
  __shared__ float thr_s;
  __shared__ uint64_t cand[LP_CAP];
  __shared__ uint64_t red[LP_THREADS / 32];
  __shared__ int count;
  if (split > 1) cluster_arrive_relaxed();  // this CTA has started; waited for before the first remote store
  pdl_enter();
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5;
  const int rank = split > 1 ? (int)cluster_ctarank() : 0;
  const int64_t r = blockIdx.x / split;
  const T* row = x + r * ld;
  const int c0 = (int)((int64_t)V * rank / split), c1 = (int)((int64_t)V * (rank + 1) / split);
  LpStat st{LP_LEAST, __fmul_rn(LP_LEAST, LOG2E), 0.f, 0.f};
  constexpr int U = LP_UNROLL<T>;
  auto all_of_them = [](int) { return true; };
  lp_for_each<T, U, false>(row, c0, c1, all_of_them, [&](int batch, const auto&, const auto& v) {
    const float hi = lp_add(st, v);
    if (k > 0 && batch >= 0 && batch < LP_KEPT) kept[batch * LP_THREADS + tid] = hi;
  });
  if (k > 0) {
    // the maxima of the groups of LP_THREADS / LP_GROUPS neighbouring threads
    float g = st.m;
#pragma unroll
    for (int o = LP_THREADS / LP_GROUPS / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
    if (tid % (LP_THREADS / LP_GROUPS) == 0) gmax[tid / (LP_THREADS / LP_GROUPS)] = g;
  }
  // the CTA's maximum, then the sums about it
  float hi = st.m;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
  if (lane == 0) wmax[wp] = hi;
  if (tid == 0) count = 0;
  __syncthreads();
#pragma unroll
  for (int w = 0; w < LP_THREADS / 32; ++w) hi = fmaxf(hi, wmax[w]);
  st.raise(hi);
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    st.s += __shfl_xor_sync(0xffffffffu, st.s, o);
    st.u += __shfl_xor_sync(0xffffffffu, st.u, o);
  }
  if (lane == 0) wsum[wp] = make_float2(st.s, st.u);
  __syncthreads();
  if (split > 1) cluster_wait_acquire();  // the first CTA's shared memory is there
  if (tid == 0) {
    LpStat all{st.m, st.m2, 0.f, 0.f};
#pragma unroll
    for (int w = 0; w < LP_THREADS / 32; ++w) {
      all.s += wsum[w].x;
      all.u += wsum[w].y;
    }
    if (rank == 0) {
      runs[0] = all;
    } else {
      const uint32_t to = mapa_shared(smem_u32(&runs[rank]), 0);
      asm volatile("st.shared::cluster.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(to), "f"(all.m), "f"(all.m2), "f"(all.s),
                   "f"(all.u)
                   : "memory");
    }
  }
  if (k > 0) {
    auto give = [&](int place, uint64_t key) {
      const uint32_t to = mapa_shared(smem_u32(&best[rank * k + place]), 0);
      asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(to), "l"(key) : "memory");
    };
    if (tid < LP_GROUPS) {
      int place = 0;
      const float mine = gmax[tid];
#pragma unroll
      for (int j = 0; j < LP_GROUPS; j += 4) {
        const float4 g = *reinterpret_cast<const float4*>(gmax + j);
        place += (g.x > mine || (g.x == mine && j < tid)) + (g.y > mine || (g.y == mine && j + 1 < tid)) +
                 (g.z > mine || (g.z == mine && j + 2 < tid)) + (g.w > mine || (g.w == mine && j + 3 < tid));
      }
      if (place == k - 1) thr_s = mine;
    }
    __syncthreads();
    // below -1e30 there is no threshold: fewer than k groups hold a logit that is not masked. Those
    // above it are then taken, and masked ones in the order of their ids where they are fewer than k.
    const float thr = thr_s;
    const bool few = thr <= LP_LEAST;
    auto reaches = [&](float v) { return few ? !(v <= thr) : !(v < thr); };
    auto want = [&](int batch) { return batch >= LP_KEPT || reaches(kept[batch * LP_THREADS + tid]); };
    lp_for_each<T, U, true>(row, c0, c1, want, [&](int, const auto& ids, const auto& v) {
      constexpr int NV = (int)(sizeof(v) / sizeof(float)), NI = (int)(sizeof(ids) / sizeof(int));
#pragma unroll
      for (int i = 0; i < NV; ++i) {
        if (reaches(v[i])) {
          const int at = atomicAdd(&count, 1);
          if (at < LP_CAP) cand[at] = lp_key(v[i], (uint32_t)(ids[i / (NV / NI)] + i % (NV / NI)));
        }
      }
    });
    __syncthreads();
    const int n = count;
    if (n <= LP_CAP && (n >= k || !few)) {
      // each candidate's place is the number of better ones (above a threshold there are k at least)
      for (int c = tid; c < n; c += LP_THREADS) {
        const uint64_t key = cand[c];
        int place = 0;
#pragma unroll 8
        for (int j = 0; j < n; ++j) place += cand[j] > key ? 1 : 0;
        if (place < k) give(place, key);
      }
    } else {
      // more equal logits than the list holds, or too few that are not masked: the best one after the
      // last, k times
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        uint64_t top = 0;
        lp_for_each<T, U, true>(row, c0, c1, all_of_them, [&](int, const auto& ids, const auto& v) {
          constexpr int NV = (int)(sizeof(v) / sizeof(float)), NI = (int)(sizeof(ids) / sizeof(int));
#pragma unroll
          for (int i = 0; i < NV; ++i) {
            const uint64_t key = lp_key(v[i], (uint32_t)(ids[i / (NV / NI)] + i % (NV / NI)));
            if (key < last && key > top) top = key;
          }
        });
        top = lp_block_max(top, red);
        if (tid == 0) give(j, top);
        last = top;
      }
    }
  }
  if (split > 1) cluster_sync_all(); else __syncthreads();
  if (rank != 0) return;
  LpStat all = runs[0];
  for (int i = 1; i < split; ++i) all = lp_merge(all, runs[i]);
  // logp = (x - m) - logs: log s, and how far m2 is from m log2 e. A row below -1e30 throughout leaves the sum
  // about -1e30 empty, and one of 1e38 and more may have no m2: their sums are taken anew about the maximum.
  float base = all.m, logs = logf(all.s) + fmaf(-all.m, LOG2E, all.m2) * LN2, ent = logf(all.s) - LN2 * (all.u / all.s);
  if (all.s == 0.f || (all.m >= 1e38f && all.m < INFINITY)) {
    float hi = -INFINITY;
    for (int c = tid; c < V; c += LP_THREADS) hi = fmaxf(hi, lp_load(row + c));
    const float top = lp_key_value(lp_block_max(lp_key(hi, 0), red));
    double s = 0.0, u = 0.0;
    for (int c = tid; c < V; c += LP_THREADS) {
      const double d = (double)lp_load(row + c) - (double)top, e = exp(d);
      s += e;
      if (e > 0.0) u += e * d;
    }
    __shared__ double dred[2][LP_THREADS / 32];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      s += __shfl_xor_sync(0xffffffffu, s, o);
      u += __shfl_xor_sync(0xffffffffu, u, o);
    }
    if (lane == 0) {
      dred[0][wp] = s;
      dred[1][wp] = u;
    }
    __syncthreads();
    s = u = 0.0;
#pragma unroll
    for (int w = 0; w < LP_THREADS / 32; ++w) {
      s += dred[0][w];
      u += dred[1][w];
    }
    base = top;
    logs = (float)log(s);  // NaN for a row of -inf alone
    ent = (float)(log(s) - u / s);
  }
  if (tid == 0) {
    logprobs[r] = lp_given(row, tokens[r], V, base, logs);
    entropy[r] = ent;
    if (stats) {
      stats[2 * r] = base;
      stats[2 * r + 1] = logs;
    }
  }
  const int n = split * k;
  for (int c = tid; c < n; c += LP_THREADS) {
    const uint64_t key = best[c];
    int place = 0;
    for (int j = 0; j < n; ++j) place += best[j] > key ? 1 : 0;
    if (place < k) {
      top_ids[r * k + place] = lp_key_id(key);
      top_logprobs[r * k + place] = (lp_key_value(key) - base) - logs;
    }
  }
}

template <typename T>
__device__ __forceinline__ void lp_store(T* p, float v);
template <>
__device__ __forceinline__ void lp_store<float>(float* p, float v) {
  *p = v;
}
template <>
__device__ __forceinline__ void lp_store<__nv_bfloat16>(__nv_bfloat16* p, float v) {
  *p = __float2bfloat16_rn(v);
}

// Elementwise: CTA (row, run of LP_BWD_RUN columns). 16-byte pieces where both rows have the same place
// in theirs, else one logit at a time. Bound by HBM (read and write; 4096 x 32000 bf16: 86 us, 6.1 TB/s).
constexpr int LP_BWD_RUN = 16384;
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
    lp_rows_bwd_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens,
                       const float* __restrict__ stats, const float* __restrict__ entropy,
                       const float* __restrict__ dlogprobs, const float* __restrict__ dentropy,
                       T* __restrict__ dx, int64_t ld_dx, int V) {
  pdl_enter();
  constexpr int NV = LpVec<T>::N, U = 4;
  const int64_t r = blockIdx.x;
  const LpCoef c = lp_coef(tokens, stats, entropy, dlogprobs, dentropy, r, V);
  const int c0 = blockIdx.y * LP_BWD_RUN, n = min(LP_BWD_RUN, V - c0), tid = threadIdx.x;
  const T* src = x + r * ld + c0;
  T* dst = dx + r * ld_dx + c0;
  const bool same = ((reinterpret_cast<uintptr_t>(src) ^ reinterpret_cast<uintptr_t>(dst)) & 15) == 0;
  const int head = same ? lp_head(src, n) : n, nvec = (n - head) / NV;
#pragma unroll 4
  for (int i = tid; i < head; i += LP_THREADS) lp_store(dst + i, c.others(lp_load(src + i)));
  const uint4* sv = reinterpret_cast<const uint4*>(src + head);
  uint4* dv = reinterpret_cast<uint4*>(dst + head);
  auto piece = [&](const uint4& q, int i) {
    float v[NV];
    LpVec<T>::unpack(q, v);
#pragma unroll
    for (int j = 0; j < NV; j += 2) c.others2(v[j], v[j + 1]);
    dv[i] = LpVec<T>::pack(v);
  };
  int i = tid;
  for (; i + (U - 1) * LP_THREADS < nvec; i += U * LP_THREADS) {
    uint4 q[U];
#pragma unroll
    for (int j = 0; j < U; ++j) q[j] = sv[i + j * LP_THREADS];
#pragma unroll
    for (int j = 0; j < U; ++j) piece(q[j], i + j * LP_THREADS);
  }
  for (; i < nvec; i += LP_THREADS) piece(sv[i], i);
  const int tail = head + nvec * NV + tid;
  if (tail < n) lp_store(dst + tail, c.others(lp_load(src + tail)));
  __syncthreads();
  if (tid == 0 && c.t >= c0 && c.t < c0 + n) lp_store(dst + (c.t - c0), c.others(lp_load(src + (c.t - c0))) + c.a);
}

int lp_sms() {
  const int dev = current_device();
  return dev >= 0 ? sm_count(dev) : 148;
}

// A row is split over as many CTAs as fit on the GPU at once, each with 2048 logits at
// least.
int lp_rows_fwd(const void* x, int dtype, int64_t ld, const int64_t* tokens, float* logprobs, float* entropy,
                float* stats, int64_t* top_ids, float* top_logprobs, int64_t N, int64_t V, int k, cudaStream_t st) {
  int split = 1;
  const int ctas = dtype == ULM_F32 ? LP_CTAS<float> : LP_CTAS<__nv_bfloat16>;
  while (split < LP_MAX_SPLIT && N * split * 2 <= ctas * (int64_t)lp_sms() && V / (split * 2) >= 2048) split *= 2;
  ULM_REQUIRE(N * split < (1ll << 31), "extent too large");
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3((unsigned)(N * split));
  cfg.blockDim = dim3(LP_THREADS);
  cfg.stream = st;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = pdl_enabled();
  attr[1].id = cudaLaunchAttributeClusterDimension;
  attr[1].val.clusterDim.x = (unsigned)split;
  attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 2;
  if (dtype == ULM_F32)
    ULM_CUDA_TRY(cudaLaunchKernelEx(&cfg, lp_rows_kernel<float>, static_cast<const float*>(x), ld, tokens, logprobs, entropy,
                                    stats, top_ids, top_logprobs, (int)V, k, split));
  else
    ULM_CUDA_TRY(cudaLaunchKernelEx(&cfg, lp_rows_kernel<__nv_bfloat16>, static_cast<const __nv_bfloat16*>(x), ld, tokens,
                                    logprobs, entropy, stats, top_ids, top_logprobs, (int)V, k, split));
  return ULM_OK;
}

template <typename T>
int lp_rows_bwd(const void* x, int64_t ld, const int64_t* tokens, const float* stats, const float* entropy,
                const float* dlogprobs, const float* dentropy, void* dx, int64_t ld_dx, int64_t N, int64_t V,
                cudaStream_t st) {
  const int64_t runs = cdiv(V, LP_BWD_RUN);
  ULM_REQUIRE(runs < 65536, "extent too large");
  return launch_pdl(lp_rows_bwd_kernel<T>, dim3((unsigned)N, (unsigned)runs), dim3(LP_THREADS), 0, st,
                    static_cast<const T*>(x), ld, tokens, stats, entropy, dlogprobs, dentropy, static_cast<T*>(dx), ld_dx,
                    (int)V);
}

// out = the sum of `parts` arrays of n, in order; four values a thread where all starts allow it
__global__ void __launch_bounds__(256)
    lp_add_kernel(const float* __restrict__ part, int parts, int64_t n, void* __restrict__ out, int dtype) {
  pdl_enter();
  const int64_t i0 = (int64_t)blockIdx.x * 256 + threadIdx.x, step = (int64_t)gridDim.x * 256;
  auto store = [&](int64_t i, float v) {
    if (dtype == ULM_F32)
      static_cast<float*>(out)[i] = v;
    else
      static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(v);
  };
  if (n % 4 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0) {
    for (int64_t i = i0; i < n / 4; i += step) {
      float4 s = reinterpret_cast<const float4*>(part)[i];
#pragma unroll 4
      for (int p = 1; p < parts; ++p) {
        const float4 v = reinterpret_cast<const float4*>(part + p * n)[i];
        s = make_float4(s.x + v.x, s.y + v.y, s.z + v.z, s.w + v.w);
      }
      if (dtype == ULM_F32) {
        reinterpret_cast<float4*>(out)[i] = s;
      } else {
        const __nv_bfloat162 a = __floats2bfloat162_rn(s.x, s.y), b = __floats2bfloat162_rn(s.z, s.w);
        reinterpret_cast<uint2*>(out)[i] =
            make_uint2(*reinterpret_cast<const uint32_t*>(&a), *reinterpret_cast<const uint32_t*>(&b));
      }
    }
    return;
  }
  for (int64_t i = i0; i < n; i += step) {
    float s = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) s += part[p * n + i];
    store(i, s);
  }
}

int lp_check(const int64_t* tokens, int64_t N, int64_t V) {
  ULM_REQUIRE(N >= 0 && V > 0, "bad extents N=%lld V=%lld", (long long)N, (long long)V);
  ULM_REQUIRE(N < (1ll << 31) && V < (1 << 30), "extent too large");
  ULM_REQUIRE(N == 0 || tokens, "null tokens");
  return ULM_OK;
}

int lp_check_top(int64_t N, int64_t V, int k, const int64_t* top_ids, const float* top_logprobs) {
  ULM_REQUIRE(k >= 0 && k <= LP_MAX_TOP && k <= V, "top_k=%d must be in 0 .. min(V, %d)", k, LP_MAX_TOP);
  ULM_REQUIRE(N == 0 || k == 0 || (top_ids && top_logprobs), "top_k > 0 needs top_ids and top_logprobs");
  return ULM_OK;
}

bool lp_dtype_ok(int dt) { return dt == ULM_F32 || dt == ULM_BF16; }

constexpr int LP_MAX_K_SPLITS = 32;

// bf16 parts of the logits' gradient in bf16 precision: two hold 16 of its digits (2^-17 of each value), so
// that dh and dW have the error of their own rounding (0.0017 in bf16). One part rounds each value by up to
// 2^-8 on the way (an error of 0.0024 to 0.0033, the more the fewer entries carry a row), and what rounding
// adds to a row no longer sums to zero as the softmax's gradient does. The second part costs another pass of
// both products and 2 bytes a logit (V = 32000, D = 768, backward: 512 rows 101 -> 140 us, 1024 142 -> 231,
// 8192 920 -> 1705).
constexpr int LP_PARTS = 2;
constexpr int64_t LP_DUMP_BYTES = 256ll << 20;

// How the head's forward finds the alternatives: from register lists of chunks where the rows are so many
// for k that the epilogue sees a row long enough to keep its list for most chunks, or from the logits
// themselves, written out for as many rows at a time as 256 MB hold. Lists against written out at V = 32000,
// D = 768, us: k = 1, 1024 rows 51 and 63 (333 rows x 288: 30 and 29); k = 8, 1024 rows 80 and 65, 2048 116
// and 119, 4096 185 and 245; k = 20, 4096 rows 294 and 265, 8192 520 and 555; k = 32, 8192 rows 630 and 570,
// 16384 1075 and 1177.
bool lp_lists(int64_t N, int64_t V, int k) { return k > 0 && N * V > 320ll * k * 32000; }
int64_t lp_ld_max(int64_t V) { return cdiv(V, 256) * 8; }  // chunks of whole tiles
int64_t lp_rows_at_once(int64_t N, int64_t V, int k) {
  if (k == 0 || lp_lists(N, V, k)) return N;
  const int64_t fit = std::max<int64_t>(1, (LP_DUMP_BYTES / (lp_ld_max(V) * 128)) / 256) * 256;
  // even steps
  return std::min(N, cdiv(cdiv(N, cdiv(N, fit)), 256) * 256);
}

// Ranges of k into which the product (rows x D) over k of the backward is split.
//
// The tensor cores cut off what an accumulator cannot hold, a little with each step of 16 in k, always
// towards zero: fp32 products are taken over ranges of about 256, as far as `room` floats hold their sums,
// which are added with rounding (at 1001 x 4099 x 288 the gradients' error falls from 8e-6 to 5e-7; ranges
// of 512 have 1e-6 and take 95 instead of 101 us there, 73 instead of 65 at 16 x 1416 x 768).
//
// A bf16 product whose 256 x 256 tiles fill the CTA pairs badly (8192 x 768: 96 tiles, two rounds of 74) is
// split where the rounds saved are worth writing and adding the partial sums (one part of that one over
// 32000: 346 us, split in three 260 + 15).
int lp_splits(int64_t rows, int64_t k, int64_t D, bool f32, int64_t room) {
  int splits = 1;
  if (f32) {
    splits = (int)std::min<int64_t>(room / std::max<int64_t>(1, rows * D), cdiv(k, 256));
  } else {
    const int pairs = lp_sms() / 2;
    const int64_t tiles = cdiv(rows, 256) * cdiv(D, 256);
    const double round_us = 2.0 * 256 * 256 * (double)k * LP_PARTS / 19e6;  // of all pairs, at 1400 TFLOP/s
    const double part_us = (double)rows * (double)D * 8 / 6.5e6;            // a partial sum, written and read
    double least = (double)cdiv(tiles, pairs) * round_us;
    for (int c = 2; c <= LP_MAX_K_SPLITS && c * 512 <= k; ++c) {
      const double t = (double)cdiv(tiles * c, pairs) / c * round_us + c * part_us + 5.0;
      if (t < least) {
        least = t;
        splits = c;
      }
    }
  }
  return splits > 1 ? (int)cdiv(k, ksplit_chunk((int)k, splits)) : 1;  // no empty range
}

// Rows of partial sums of that product: none where it is not split.
int64_t lp_sum_rows(int64_t rows, int64_t k, int64_t D, bool f32, int64_t room) {
  const int splits = lp_splits(rows, k, D, f32, room);
  return splits > 1 ? splits * rows : 0;
}

// Floats for an fp32 product's sums: 64 MB of them, or the place of the fp32 gradient of the logits, which
// its parts have replaced by then, where that is larger (that place alone would hold too few of them where the
// vocabulary is little wider than the model: 16 x 1416 x 768 107 us and an error of 2.7e-6, now 65 and 5e-7;
// 1000 x 1500 x 1024 146 and 2.9e-6, now 117 and 5e-7).
constexpr int64_t LP_SUMS = 16ll << 20;
int64_t lp_room(int64_t N, int64_t V) { return std::max(N * ulm_operand_ld(V), LP_SUMS); }

// The work buffer of the head's entries.
struct LpWork {
  void *h_parts, *w_parts, *dx, *dx_parts;
  float *part, *given, *dump, *chunk_max, *sums;
  float2* list;
  int64_t bytes;
};
LpWork lp_work(void* base, int64_t N, int64_t V, int64_t D, int k, bool backward, bool f32) {
  char* p = static_cast<char*>(base);
  auto take = [&](int64_t bytes) {
    char* q = p;
    p += (bytes + 255) / 256 * 256;
    return q;
  };
  auto floats = [&](int64_t n) { return reinterpret_cast<float*>(take(n * 4)); };
  LpWork w{};
  const int64_t ldd = ulm_operand_ld(D), ldv = ulm_operand_ld(V);
  if (f32) {
    w.h_parts = take(3 * N * ldd * 2);
    w.w_parts = take(3 * V * ldd * 2);
  }
  if (backward) {
    w.dx = take(N * ldv * (f32 ? 4 : 2 * LP_PARTS));
    if (f32) w.dx_parts = take(3 * N * ldv * 2);
    // partial sums of dh, then of dW
    const int64_t room = lp_room(N, V);
    if (f32 && room > LP_SUMS)
      w.sums = static_cast<float*>(w.dx);
    else
      w.sums = floats(std::max(lp_sum_rows(N, V, D, f32, room), lp_sum_rows(V, N, D, f32, room)) * D);
  } else {
    const int64_t rows = lp_rows_at_once(N, V, k);
    // the shares of the rows of one launch: all of them, but for the last one's fewer rows
    int64_t shares = 0;
    for (const int64_t n : {rows, N % rows}) {
      if (n == 0) continue;
      const LpShape s = lp_shape(n, V, D, f32, lp_sms());
      shares = std::max(shares, n * lp_groups(s) * s.slots * 2);
    }
    w.part = floats(shares * 4);
    w.given = floats(rows);
    if (lp_lists(N, V, k)) {
      w.list = reinterpret_cast<float2*>(take(shares * k * 8));
      w.dump = floats(shares * k * 32);
    } else if (k > 0) {
      w.dump = floats(rows * lp_ld_max(V) * 32);
      w.chunk_max = floats(rows * lp_ld_max(V));
    }
  }
  w.bytes = p - static_cast<char*>(base);
  return w;
}

int lp_head_check(const void* h_op, int64_t ld_h, const void* w_op, int64_t ld_w, const int64_t* tokens, int64_t N,
                  int64_t V, int64_t D, int prec) {
  ULM_REQUIRE(prec == ULM_PREC_BF16 || prec == ULM_PREC_FP32, "prec must be ULM_PREC_BF16 or ULM_PREC_FP32");
  if (int rc = lp_check(tokens, N, V)) return rc;
  ULM_REQUIRE(D > 0 && D < (1 << 30), "bad extent D=%lld", (long long)D);
  ULM_REQUIRE(N == 0 || (h_op && w_op), "null pointer argument");
  ULM_REQUIRE(ld_h >= D && ld_w >= D, "row stride shorter than the row");
  return ULM_OK;
}

}  // namespace
}  // namespace ulm

using namespace ulm;

extern "C" int ulm_token_logprobs_fwd(const void* logits, int dtype, int64_t ld, const int64_t* tokens,
                                      float* logprobs, float* entropy, float* stats, int64_t* top_ids,
                                      float* top_logprobs, int64_t N, int64_t V, int top_k, void* stream) {
  if (int rc = lp_check(tokens, N, V)) return rc;
  if (int rc = lp_check_top(N, V, top_k, top_ids, top_logprobs)) return rc;
  ULM_REQUIRE(lp_dtype_ok(dtype), "bad dtype");
  ULM_REQUIRE(ld >= V, "row stride shorter than the row");
  if (N == 0) return ULM_OK;
  ULM_REQUIRE(logits && logprobs && entropy, "null pointer argument");
  return lp_rows_fwd(logits, dtype, ld, tokens, logprobs, entropy, stats, top_ids, top_logprobs, N, V, top_k,
                     static_cast<cudaStream_t>(stream));
}

extern "C" int ulm_token_logprobs_bwd(const float* dlogprobs, const float* dentropy, const void* logits, int dtype,
                                      int64_t ld, const int64_t* tokens, const float* stats, const float* entropy,
                                      void* dlogits, int64_t ld_d, int64_t N, int64_t V, void* stream) {
  if (int rc = lp_check(tokens, N, V)) return rc;
  ULM_REQUIRE(lp_dtype_ok(dtype), "bad dtype");
  ULM_REQUIRE(ld >= V && ld_d >= V, "row stride shorter than the row");
  if (N == 0) return ULM_OK;
  ULM_REQUIRE(logits && stats && entropy && dlogits, "null pointer argument");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  return dtype == ULM_F32 ? lp_rows_bwd<float>(logits, ld, tokens, stats, entropy, dlogprobs, dentropy, dlogits, ld_d, N,
                                               V, st)
                          : lp_rows_bwd<__nv_bfloat16>(logits, ld, tokens, stats, entropy, dlogprobs, dentropy, dlogits,
                                                       ld_d, N, V, st);
}

extern "C" int64_t ulm_lm_head_logprobs_work_bytes(int64_t N, int64_t V, int64_t D, int top_k, int backward, int prec) {
  if (N < 0 || V <= 0 || D <= 0 || top_k < 0 || top_k > LP_MAX_TOP) return -1;
  if (N == 0) return 256;
  return lp_work(nullptr, N, V, D, top_k, backward != 0, prec == ULM_PREC_FP32).bytes;
}

extern "C" int ulm_lm_head_logprobs_fwd(const void* h_op, int64_t ld_h, const void* w_op, int64_t ld_w,
                                        const int64_t* tokens, float* logprobs, float* entropy, float* stats,
                                        int64_t* top_ids, float* top_logprobs, void* work, int64_t N, int64_t V,
                                        int64_t D, int top_k, int prec, void* stream) {
  if (int rc = lp_head_check(h_op, ld_h, w_op, ld_w, tokens, N, V, D, prec)) return rc;
  if (int rc = lp_check_top(N, V, top_k, top_ids, top_logprobs)) return rc;
  if (N == 0) return ULM_OK;
  ULM_REQUIRE(logprobs && entropy && work, "null pointer argument");
  ULM_REQUIRE(is_aligned16(work), "work must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f32 = prec == ULM_PREC_FP32;
  const LpWork w = lp_work(work, N, V, D, top_k, false, f32);
  const bool lists = lp_lists(N, V, top_k), dump = top_k > 0 && !lists;
  const int64_t step = lp_rows_at_once(N, V, top_k), es = f32 ? 4 : 2;
  CUtensorMap th, tw, to;
  memset(&to, 0, sizeof(to));
  if (int rc = lp_operand(&tw, w_op, ld_w, V, D, f32, w.w_parts, st)) return rc;
  for (int64_t r0 = 0; r0 < N; r0 += step) {
    const int64_t n = std::min(step, N - r0);
    const LpShape s = lp_shape(n, V, D, f32, lp_sms());
    const int shares = lp_groups(s) * s.slots * 2;  // of a row
    ULM_REQUIRE(shares <= LP_JOIN_MAX, "too many column groups");
    if (int rc = lp_operand(&th, static_cast<const char*>(h_op) + r0 * ld_h * es, ld_h, n, D, f32, w.h_parts, st)) return rc;
    if (dump)
      ULM_REQUIRE(make_epi_tmap(&to, EPI_MODE_WARP, w.dump, ULM_F32, V, n, 1, lp_ld_max(V) * 32, 0),
                  "no tensor map of the logits");
    LpArgs a{};
    a.tokens = tokens + r0;
    a.part = w.part;
    a.list = w.list;
    a.dump = w.dump;
    a.given = w.given;
    a.k = lists ? top_k : 0;
    a.groups = lp_groups(s);
    a.chunk_max = w.chunk_max;
    a.ld_max = lp_ld_max(V);
    if (int rc = dump    ? lp_launch<LP_DUMP, 0, false>(th, tw, to, s, a, st)
                 : !lists ? lp_launch<LP_STATS, 0, false>(th, tw, to, s, a, st)
                 : top_k <= LP_LIST ? lp_launch<LP_STATS, LP_LIST, false>(th, tw, to, s, a, st)
                                    : lp_launch<LP_STATS, LP_LONG_LIST, false>(th, tw, to, s, a, st))
      return rc;
    a.k = top_k;
    const int room = top_k == 0 ? 0 : lp_join_room(lists ? shares : 0, top_k);
    const bool wide = dump || n <= 4 * (int64_t)lp_sms();
    const int rc = launch_pdl(dump ? lp_join_kernel<128, true> : wide ? lp_join_kernel<128, false> : lp_join_kernel<32, false>,
                              dim3((unsigned)(wide ? n : cdiv(n, LP_JOIN_ROWS))), dim3(wide ? 128 : 32 * LP_JOIN_ROWS),
                              (size_t)room * 12 * (wide ? 1 : LP_JOIN_ROWS), st, s, a, logprobs + r0, entropy + r0,
                              stats ? stats + 2 * r0 : nullptr, top_ids ? top_ids + r0 * top_k : nullptr,
                              top_logprobs ? top_logprobs + r0 * top_k : nullptr, room);
    if (rc) return rc;
  }
  return ULM_OK;
}

extern "C" int ulm_lm_head_logprobs_bwd(const float* dlogprobs, const float* dentropy, const void* h_op, int64_t ld_h,
                                        const void* w_op, int64_t ld_w, const int64_t* tokens, const float* stats,
                                        const float* entropy, void* dh, int dh_dtype, void* dw, int dw_dtype,
                                        void* work, int64_t N, int64_t V, int64_t D, int prec, void* stream) {
  if (int rc = lp_head_check(h_op, ld_h, w_op, ld_w, tokens, N, V, D, prec)) return rc;
  ULM_REQUIRE(lp_dtype_ok(dh_dtype) && lp_dtype_ok(dw_dtype), "bad dtype");
  ULM_REQUIRE(N == 0 || (stats && entropy && work), "null pointer argument");
  ULM_REQUIRE(N == 0 || is_aligned16(work), "work must be 16-byte aligned");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  if (!dh && !dw) return ULM_OK;
  if (N == 0) {
    if (dw) ULM_CUDA_TRY(cudaMemsetAsync(dw, 0, V * D * (dw_dtype == ULM_F32 ? 4 : 2), st));
    return ULM_OK;
  }
  const bool f32 = prec == ULM_PREC_FP32;
  const int64_t ldv = ulm_operand_ld(V), ldd = ulm_operand_ld(D);
  const LpShape s = lp_shape(N, V, D, f32, lp_sms());
  const LpWork w = lp_work(work, N, V, D, 0, true, f32);
  CUtensorMap th, tw, to;
  if (int rc = lp_operand(&th, h_op, ld_h, N, D, f32, w.h_parts, st)) return rc;
  if (int rc = lp_operand(&tw, w_op, ld_w, V, D, f32, w.w_parts, st)) return rc;
  const int parts = f32 ? 1 : LP_PARTS;
  ULM_REQUIRE(make_epi_tmap(&to, EPI_MODE_WARP, w.dx, f32 ? ULM_F32 : ULM_BF16, V, N, parts, ldv, N * ldv),
              "no tensor map of the logits' gradient");
  LpArgs a{};
  a.tokens = tokens;
  a.stats = stats;
  a.entropy = entropy;
  a.dlogprobs = dlogprobs;
  a.dentropy = dentropy;
  if (int rc = f32 ? lp_launch<LP_GRAD, 0, true>(th, tw, to, s, a, st) : lp_launch<LP_GRAD, 0, false>(th, tw, to, s, a, st))
    return rc;
  const void *dx = w.dx, *hh = h_op, *ww = w_op;
  if (f32) {
    if (int rc = lp_split(static_cast<const float*>(w.dx), ldv, w.dx_parts, ldv, N, V, st)) return rc;
    dx = w.dx_parts;
    hh = w.h_parts;
    ww = w.w_parts;
    ld_h = ld_w = ldd;
  }
  // each product's operands are single matrices, or the parts of one (its batches)
  auto product = [&](const Operand& A, const Operand& B, int64_t rows, int64_t k, void* out, int dtype) -> int {
    GemmShape g{1, (int)rows, (int)D, (int)k, CAUSAL_NONE};
    g.parts = f32 ? 6 : LP_PARTS;
    const int splits = lp_splits(rows, k, D, f32, lp_room(N, V));
    if (splits <= 1) return run_gemm(A, B, g, make_epilogue(EPI_STORE, dtype, out, D, rows * D, nullptr), st);
    g.batches = g.ksplit = splits;
    if (int rc = run_gemm(A, B, g, make_epilogue(EPI_STORE, ULM_F32, w.sums, D, rows * D, nullptr), st)) return rc;
    return launch_pdl(lp_add_kernel, dim3((unsigned)std::min<int64_t>(cdiv(rows * D, 1024), 1 << 20)), dim3(256), 0, st,
                      static_cast<const float*>(w.sums), splits, rows * D, out, dtype);
  };
  if (dh) {
    // dh = dx W: A = dx (rows, K-major over the vocabulary), B = W as [token][d] (MN-major)
    const Operand A{dx, ldv, N * ldv, V, N, ULM_BF16, false}, Bw{ww, ld_w, V * ld_w, D, V, ULM_BF16, true};
    if (int rc = product(A, Bw, N, V, dh, dh_dtype)) return rc;
  }
  if (!dw) return ULM_OK;
  // dW = dx^T h: A = dx as [row][token] (MN-major), B = h as [row][d] (MN-major)
  const Operand A{dx, ldv, N * ldv, V, N, ULM_BF16, true}, Bh{hh, ld_h, N * ld_h, D, N, ULM_BF16, true};
  return product(A, Bh, V, N, dw, dw_dtype);
}
