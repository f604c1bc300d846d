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
constexpr int LP_CAP = 512;       // candidates of one row above the threshold

// Running statistics of a set of logits: the maximum m (-inf for none), s = sum exp(x - m) and
// u = sum exp(x - m) (x - m), taken about 0 while m is -inf (every term is then zero, or NaN).
struct LpStat {
  float m, s, u;
};

__device__ __forceinline__ LpStat lp_merge(const LpStat& a, const LpStat& b) {
  const float M = fmaxf(a.m, b.m);
  auto part = [M](const LpStat& p, float& s, float& u) {
    const float d = p.m == -INFINITY ? 0.f : p.m - M;
    const float f = fast_exp2(d * LOG2E);
    s = p.s * f;
    u = f > 0.f ? (p.u + p.s * d) * f : 0.f;
  };
  float sa, ua, sb, ub;
  part(a, sa, ua);
  part(b, sb, ub);
  return LpStat{M, sa + sb, ua + ub};
}

// NV more logits into a thread's statistics. fmaxf on the factor of u keeps exp(-inf) * -inf at 0.
template <int NV>
__device__ __forceinline__ void lp_add(LpStat& st, const float (&x)[NV]) {
  float lm = x[0];
#pragma unroll
  for (int i = 1; i < NV; ++i) lm = fmaxf(lm, x[i]);
  if (lm > st.m) {
    const float d = st.m == -INFINITY ? 0.f : st.m - lm;
    const float f = fast_exp2(d * LOG2E);
    st.u = f > 0.f ? (st.u + st.s * d) * f : 0.f;
    st.s *= f;
    st.m = lm;
  }
  const float base = st.m == -INFINITY ? 0.f : st.m;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const float d = x[i] - base;
    const float e = fast_exp2(d * LOG2E);
    st.s += e;
    st.u = fmaf(e, fmaxf(d, -1e4f), st.u);
  }
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

// Logits of 16 bytes as floats.
template <typename T>
struct LpVec;
template <>
struct LpVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[4]) {
    x[0] = __uint_as_float(q.x);
    x[1] = __uint_as_float(q.y);
    x[2] = __uint_as_float(q.z);
    x[3] = __uint_as_float(q.w);
  }
};
template <>
struct LpVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[8]) {
    const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      x[2 * i] = __uint_as_float(w[i] << 16);
      x[2 * i + 1] = __uint_as_float(w[i] & 0xFFFF0000u);
    }
  }
};

// Elements before the first 16-byte boundary of a row, at most n.
template <typename T>
__device__ __forceinline__ int lp_head(const T* row, int n) {
  const int h = (int)(((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / sizeof(T));
  return h < n ? h : n;
}

// f(id, values) over the row's V logits, 16 bytes at a time from its first 16-byte boundary, and one
// at a time at the two ends; thread t takes every LP_THREADS-th piece.
template <typename T, typename F1, typename FV>
__device__ __forceinline__ void lp_for_each(const T* row, int V, F1&& one, FV&& vec) {
  constexpr int NV = LpVec<T>::N;
  const int head = lp_head(row, V), nvec = (V - head) / NV, tail0 = head + nvec * NV;
  const uint4* body = reinterpret_cast<const uint4*>(row + head);
  if ((int)threadIdx.x < head) one((int)threadIdx.x, lp_load(row + threadIdx.x));
#pragma unroll 4
  for (int i = threadIdx.x; i < nvec; i += LP_THREADS) {
    float x[NV];
    LpVec<T>::unpack(body[i], x);
    vec(head + i * NV, x);
  }
  if (tail0 + (int)threadIdx.x < V) one(tail0 + (int)threadIdx.x, lp_load(row + tail0 + threadIdx.x));
}

// The row's logp of its token from its statistics.
template <typename T>
__device__ __forceinline__ float lp_given(const T* row, int64_t t, int V, float base, float logs) {
  if (t == -1) return 0.f;
  if (t < 0 || t >= V) return __uint_as_float(0x7FC00000u);
  return (lp_load(row + t) - base) - logs;
}

// One CTA per row.
template <typename T>
__global__ void __launch_bounds__(LP_THREADS)
    lp_rows_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens,
                   float* __restrict__ logprobs, float* __restrict__ entropy, float* __restrict__ stats,
                   int64_t* __restrict__ top_ids, float* __restrict__ top_logprobs, int V, int k) {
  __shared__ LpStat part[LP_THREADS / 32];
  __shared__ float gmax[LP_GROUPS];
  __shared__ float thr_s;
  __shared__ uint64_t cand[LP_CAP];
  __shared__ uint64_t red[LP_THREADS / 32];
  __shared__ int count;
  const int tid = threadIdx.x, lane = tid & 31, wp = tid >> 5;
  const int64_t r = blockIdx.x;
  const T* row = x + r * ld;
  LpStat st{-INFINITY, 0.f, 0.f};
  lp_for_each(
      row, V,
      [&](int, float v) {
        const float one[1] = {v};
        lp_add(st, one);
      },
      [&](int, const auto& v) { lp_add(st, v); });
  // the maxima of the groups of LP_THREADS / LP_GROUPS neighbouring threads
  float g = st.m;
#pragma unroll
  for (int o = LP_THREADS / LP_GROUPS / 2; o > 0; o >>= 1) g = fmaxf(g, __shfl_xor_sync(0xffffffffu, g, o));
  if (tid % (LP_THREADS / LP_GROUPS) == 0) gmax[tid / (LP_THREADS / LP_GROUPS)] = g;
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const LpStat other{__shfl_xor_sync(0xffffffffu, st.m, o), __shfl_xor_sync(0xffffffffu, st.s, o),
                       __shfl_xor_sync(0xffffffffu, st.u, o)};
    st = lp_merge(st, other);
  }
  if (lane == 0) part[wp] = st;
  if (tid == 0) count = 0;
  __syncthreads();
  LpStat all = part[0];
#pragma unroll
  for (int w = 1; w < LP_THREADS / 32; ++w) all = lp_merge(all, part[w]);
  const float base = all.m == -INFINITY ? 0.f : all.m;
  const float logs = logf(all.s);
  if (tid == 0) {
    logprobs[r] = lp_given(row, tokens[r], V, base, logs);
    entropy[r] = logs - all.u / all.s;
    if (stats) {
      stats[2 * r] = base;
      stats[2 * r + 1] = logs;
    }
  }
  if (k == 0) return;
  // The k-th largest group maximum bounds the k-th best logit from below: only logits not under it
  // are candidates (about k of them, unless many are equal).
  if (tid < LP_GROUPS) {
    int rank = 0;
    const float mine = gmax[tid];
#pragma unroll 8
    for (int j = 0; j < LP_GROUPS; ++j) rank += (gmax[j] > mine || (gmax[j] == mine && j < tid)) ? 1 : 0;
    if (rank == k - 1) thr_s = mine;
  }
  __syncthreads();
  const float thr = thr_s;
  auto offer = [&](int id, float v) {
    if (!(v < thr)) {
      const int at = atomicAdd(&count, 1);
      if (at < LP_CAP) cand[at] = lp_key(v, (uint32_t)id);
    }
  };
  lp_for_each(row, V, offer, [&](int id, const auto& v) {
#pragma unroll
    for (int i = 0; i < LpVec<T>::N; ++i) offer(id + i, v[i]);
  });
  __syncthreads();
  const int n = count;
  if (n <= LP_CAP) {
    // each candidate's place is the number of better ones
    for (int c = tid; c < n; c += LP_THREADS) {
      const uint64_t key = cand[c];
      int rank = 0;
      for (int j = 0; j < n; ++j) rank += cand[j] > key ? 1 : 0;
      if (rank < k) {
        top_ids[r * k + rank] = lp_key_id(key);
        top_logprobs[r * k + rank] = (lp_key_value(key) - base) - logs;
      }
    }
    return;
  }
  // many equal logits: the best one after the last, k times
  uint64_t last = ~0ull;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    auto look = [&](int id, float v) {
      const uint64_t key = lp_key(v, (uint32_t)id);
      if (key < last && key > best) best = key;
    };
    lp_for_each(row, V, look, [&](int id, const auto& v) {
#pragma unroll
      for (int i = 0; i < LpVec<T>::N; ++i) look(id + i, v[i]);
    });
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const uint64_t other = __shfl_xor_sync(0xffffffffu, best, o);
      best = other > best ? other : best;
    }
    __syncthreads();
    if (lane == 0) red[wp] = best;
    __syncthreads();
    best = red[0];
#pragma unroll
    for (int w = 1; w < LP_THREADS / 32; ++w) best = red[w] > best ? red[w] : best;
    last = best;
    if (tid == 0) {
      top_ids[r * k + j] = lp_key_id(best);
      top_logprobs[r * k + j] = (lp_key_value(best) - base) - logs;
    }
  }
}

__device__ __forceinline__ float lp_dlogit(const LpCoef& c, float x, int64_t v) {
  const float logp = (x - c.base) - c.logs;
  const float p = fast_exp2(logp * LOG2E);
  const float d = p == 0.f ? 0.f : p * (c.b != 0.f ? fmaf(c.b, logp, c.c0) : c.c0);
  return (v == c.t ? c.a : 0.f) - d;
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

template <typename T, typename TO>
__global__ void __launch_bounds__(LP_THREADS)
    lp_rows_bwd_kernel(const T* __restrict__ x, int64_t ld, const int64_t* __restrict__ tokens,
                       const float* __restrict__ stats, const float* __restrict__ entropy,
                       const float* __restrict__ dlogprobs, const float* __restrict__ dentropy,
                       TO* __restrict__ dx, int64_t ld_dx, int V) {
  const int64_t r = blockIdx.x;
  const LpCoef c = lp_coef(tokens, stats, entropy, dlogprobs, dentropy, r, V);
  for (int v = threadIdx.x; v < V; v += LP_THREADS)
    lp_store(dx + r * ld_dx + v, lp_dlogit(c, lp_load(x + r * ld + v), v));
}

int lp_rows_fwd(const void* x, int dtype, int64_t ld, const int64_t* tokens, float* logprobs, float* entropy,
                float* stats, int64_t* top_ids, float* top_logprobs, int64_t N, int64_t V, int k, cudaStream_t st) {
  if (dtype == ULM_F32)
    lp_rows_kernel<float><<<(unsigned)N, LP_THREADS, 0, st>>>(static_cast<const float*>(x), ld, tokens, logprobs, entropy,
                                                              stats, top_ids, top_logprobs, (int)V, k);
  else
    lp_rows_kernel<__nv_bfloat16><<<(unsigned)N, LP_THREADS, 0, st>>>(static_cast<const __nv_bfloat16*>(x), ld, tokens,
                                                                      logprobs, entropy, stats, top_ids, top_logprobs,
                                                                      (int)V, k);
  ULM_LAUNCH_CHECK("lp_rows_kernel");
  return ULM_OK;
}

template <typename T, typename TO>
int lp_rows_bwd_t(const void* x, int64_t ld, const int64_t* tokens, const float* stats, const float* entropy,
                  const float* dlogprobs, const float* dentropy, void* dx, int64_t ld_dx, int64_t N, int64_t V,
                  cudaStream_t st) {
  lp_rows_bwd_kernel<T, TO><<<(unsigned)N, LP_THREADS, 0, st>>>(static_cast<const T*>(x), ld, tokens, stats, entropy,
                                                                dlogprobs, dentropy, static_cast<TO*>(dx), ld_dx,
                                                                (int)V);
  ULM_LAUNCH_CHECK("lp_rows_bwd_kernel");
  return ULM_OK;
}

// out = the sum of `parts` arrays of n, in order
__global__ void __launch_bounds__(256)
    lp_add_kernel(const float* __restrict__ part, int parts, int64_t n, void* __restrict__ out, int dtype) {
  pdl_enter();
  for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
    float s = 0.f;
#pragma unroll 8
    for (int p = 0; p < parts; ++p) s += part[p * n + i];
    if (dtype == ULM_F32)
      static_cast<float*>(out)[i] = s;
    else
      static_cast<__nv_bfloat16*>(out)[i] = __float2bfloat16_rn(s);
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

int lp_sms() {
  const int dev = current_device();
  return dev >= 0 ? sm_count(dev) : 148;
}

// The work buffer of the head's entries.
struct LpWork {
  void *h_parts, *w_parts, *dx, *dx_parts;
  float *part, *given, *dump;
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
  LpWork w{};
  const int64_t ldd = ulm_operand_ld(D), ldv = ulm_operand_ld(V);
  if (f32) {
    w.h_parts = take(3 * N * ldd * 2);
    w.w_parts = take(3 * V * ldd * 2);
  }
  if (backward) {
    w.dx = take(N * ldv * (f32 ? 4 : 2));
    if (f32) w.dx_parts = take(3 * N * ldv * 2);
  } else {
    const LpShape s = lp_shape(N, V, D, f32, lp_sms());
    const int64_t shares = N * lp_groups(s) * s.slots * 2;
    w.part = reinterpret_cast<float*>(take(shares * 16));
    w.list = reinterpret_cast<float2*>(take(shares * k * 8));
    w.dump = reinterpret_cast<float*>(take(shares * k * 128));
    w.given = reinterpret_cast<float*>(take(N * 4));
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
  return dtype == ULM_F32 ? lp_rows_bwd_t<float, float>(logits, ld, tokens, stats, entropy, dlogprobs, dentropy,
                                                        dlogits, ld_d, N, V, st)
                          : lp_rows_bwd_t<__nv_bfloat16, __nv_bfloat16>(logits, ld, tokens, stats, entropy, dlogprobs,
                                                                        dentropy, dlogits, ld_d, N, V, st);
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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const bool f32 = prec == ULM_PREC_FP32;
  const LpShape s = lp_shape(N, V, D, f32, lp_sms());
  const LpWork w = lp_work(work, N, V, D, top_k, false, f32);
  ULM_REQUIRE(lp_groups(s) * s.slots * 2 <= LP_JOIN_MAX, "too many column groups");
  CUtensorMap th, tw, to;
  memset(&to, 0, sizeof(to));
  if (int rc = lp_operand(&th, h_op, ld_h, N, D, f32, w.h_parts, st)) return rc;
  if (int rc = lp_operand(&tw, w_op, ld_w, V, D, f32, w.w_parts, st)) return rc;
  LpArgs a{};
  a.tokens = tokens;
  a.part = w.part;
  a.list = w.list;
  a.dump = w.dump;
  a.given = w.given;
  a.k = top_k;
  a.groups = lp_groups(s);
  const int K = lp_list_k(top_k);
  const int rc = K == 0   ? lp_launch<LP_STATS, 0, false>(th, tw, to, s, a, st)
                 : K == 8 ? lp_launch<LP_STATS, 8, false>(th, tw, to, s, a, st)
                          : lp_launch<LP_STATS, 32, false>(th, tw, to, s, a, st);
  if (rc) return rc;
  return launch_pdl(lp_join_kernel, dim3((unsigned)cdiv(N, LP_JOIN_WARPS)), dim3(32 * LP_JOIN_WARPS), 0, st, s, a,
                    logprobs, entropy, stats, top_ids, top_logprobs);
}

extern "C" int ulm_lm_head_logprobs_bwd(const float* dlogprobs, const float* dentropy, const void* h_op, int64_t ld_h,
                                        const void* w_op, int64_t ld_w, const int64_t* tokens, const float* stats,
                                        const float* entropy, void* dh, int dh_dtype, void* dw, int dw_dtype,
                                        void* work, int64_t N, int64_t V, int64_t D, int prec, void* stream) {
  if (int rc = lp_head_check(h_op, ld_h, w_op, ld_w, tokens, N, V, D, prec)) return rc;
  ULM_REQUIRE(lp_dtype_ok(dh_dtype) && lp_dtype_ok(dw_dtype), "bad dtype");
  ULM_REQUIRE(N == 0 || (stats && entropy && work), "null pointer argument");
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
  ULM_REQUIRE(make_epi_tmap(&to, EPI_MODE_WARP, w.dx, f32 ? ULM_F32 : ULM_BF16, V, N, 1, ldv, N * ldv),
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
    const int64_t ctas = cdiv(N * ldv, 256 * 8);
    if (int rc = launch_pdl(lp_split_kernel, dim3((unsigned)(ctas < 8192 ? ctas : 8192)), dim3(256), 0, st,
                            static_cast<const float*>(w.dx), ldv, static_cast<__nv_bfloat16*>(w.dx_parts), ldv, N, V))
      return rc;
    dx = w.dx_parts;
    hh = w.h_parts;
    ww = w.w_parts;
    ld_h = ld_w = ldd;
  }
  // Each product's operands are single matrices, or the three parts of one (its batches). The tensor cores
  // cut off what an accumulator cannot hold, a little with each step of 16 in k, always towards zero: fp32
  // products are taken over ranges of about 512, whose sums are added with rounding (at 1001 x 4099 x 288
  // the gradients' error falls from 8e-6 to below 2e-6). The ranges' sums take the place of the fp32
  // gradient of the logits, which its parts have replaced.
  auto product = [&](const Operand& A, const Operand& B, int64_t rows, int64_t k, void* out, int dtype) -> int {
    GemmShape g{1, (int)rows, (int)D, (int)k, CAUSAL_NONE};
    if (!f32) return run_gemm(A, B, g, make_epilogue(EPI_STORE, dtype, out, D, rows * D, nullptr), st);
    g.parts = 6;
    const int64_t room = N * ldv / (rows * D);
    int splits = (int)std::min<int64_t>(room, cdiv(k, 512));
    if (splits > 1) splits = (int)cdiv(k, ksplit_chunk((int)k, splits));
    if (splits <= 1) return run_gemm(A, B, g, make_epilogue(EPI_STORE, dtype, out, D, rows * D, nullptr), st);
    g.batches = g.ksplit = splits;
    float* sums = static_cast<float*>(w.dx);
    if (int rc = run_gemm(A, B, g, make_epilogue(EPI_STORE, ULM_F32, sums, D, rows * D, nullptr), st)) return rc;
    return launch_pdl(lp_add_kernel, dim3((unsigned)std::min<int64_t>(cdiv(rows * D, 256), 1 << 20)), dim3(256), 0, st,
                      static_cast<const float*>(sums), splits, rows * D, out, dtype);
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
