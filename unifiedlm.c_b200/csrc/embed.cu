// Token embedding with a scale, and its weight's gradient:
//   y_n = scale * W[t_n],   dW_v = scale * sum over the positions n with t_n = v of dy_n
// The sum runs over the positions in ascending order (no atomics: the same bits in every run).
// Token -1 is padding: a zero row, no gradient. Any other token outside [0, V) gives a NaN row and
// takes no gradient (there is no row to put it in).
#include "common.cuh"

namespace ulm {
namespace {

constexpr int EMB_THREADS = 256;

__device__ __forceinline__ float emb_load(const void* p, int dtype, int64_t i) {
  return dtype == ULM_F32 ? static_cast<const float*>(p)[i]
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void emb_store(void* p, int dtype, int64_t i, float v) {
  if (dtype == ULM_F32)
    static_cast<float*>(p)[i] = v;
  else
    static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

__global__ void __launch_bounds__(EMB_THREADS)
    embedding_fwd_kernel(const int64_t* __restrict__ tokens, const void* __restrict__ w, int w_dtype, int64_t ld_w,
                         void* __restrict__ y, int y_dtype, int64_t V, int64_t D, float scale) {
  const int64_t n = blockIdx.x;
  const int64_t t = tokens[n];
  for (int64_t d = threadIdx.x; d < D; d += EMB_THREADS) {
    float v = t == -1 ? 0.f : __uint_as_float(0x7FC00000u);
    if (t >= 0 && t < V) v = emb_load(w, w_dtype, t * ld_w + d) * scale;
    emb_store(y, y_dtype, n * D + d, v);
  }
}

// One CTA per row of W: it looks through the tokens, a block at a time, and adds the rows of dy whose
// token is its own.
__global__ void __launch_bounds__(EMB_THREADS)
    embedding_bwd_kernel(const int64_t* __restrict__ tokens, const void* __restrict__ dy, int dy_dtype,
                         void* __restrict__ dw, int dw_dtype, int64_t N, int64_t D, float scale) {
  __shared__ int64_t found[EMB_THREADS];
  __shared__ int wcount[EMB_THREADS / 32];
  const int64_t v = blockIdx.x;
  const int lane = threadIdx.x & 31, wp = threadIdx.x >> 5;
  for (int64_t d0 = 0; d0 < D; d0 += 4 * EMB_THREADS) {
    float acc[4] = {0.f, 0.f, 0.f, 0.f};
    for (int64_t n0 = 0; n0 < N; n0 += EMB_THREADS) {
      const int64_t n = n0 + threadIdx.x;
      const bool hit = n < N && tokens[n] == v;
      const unsigned b = __ballot_sync(0xffffffffu, hit);
      __syncthreads();
      if (lane == 0) wcount[wp] = __popc(b);
      __syncthreads();
      int at = __popc(b & ((1u << lane) - 1u)), total = 0;
      for (int i = 0; i < EMB_THREADS / 32; ++i) {
        if (i < wp) at += wcount[i];
        total += wcount[i];
      }
      if (hit) found[at] = n;
      __syncthreads();
      for (int j = 0; j < total; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const int64_t d = d0 + i * EMB_THREADS + threadIdx.x;
          if (d < D) acc[i] += emb_load(dy, dy_dtype, found[j] * D + d);
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int64_t d = d0 + i * EMB_THREADS + threadIdx.x;
      if (d < D) emb_store(dw, dw_dtype, v * D + d, acc[i] * scale);
    }
  }
}

int emb_check(const int64_t* tokens, int64_t N, int64_t V, int64_t D) {
  ULM_REQUIRE(N >= 0 && V > 0 && D > 0, "bad extents N=%lld V=%lld D=%lld", (long long)N, (long long)V, (long long)D);
  ULM_REQUIRE(N < (1ll << 31) && V < (1ll << 31) && D < (1 << 30), "extent too large");
  ULM_REQUIRE(N == 0 || tokens, "null tokens");
  return ULM_OK;
}
bool emb_dtype_ok(int dt) { return dt == ULM_F32 || dt == ULM_BF16; }

}  // namespace
}  // namespace ulm

using namespace ulm;

extern "C" int ulm_embedding_fwd(const int64_t* tokens, const void* weight, int w_dtype, int64_t ld_w, void* y,
                                 int y_dtype, int64_t N, int64_t V, int64_t D, float scale, void* stream) {
  if (int rc = emb_check(tokens, N, V, D)) return rc;
  ULM_REQUIRE(emb_dtype_ok(w_dtype) && emb_dtype_ok(y_dtype), "bad dtype");
  ULM_REQUIRE(ld_w >= D, "row stride shorter than the row");
  if (N == 0) return ULM_OK;
  ULM_REQUIRE(weight && y, "null pointer argument");
  embedding_fwd_kernel<<<(unsigned)N, EMB_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(tokens, weight, w_dtype, ld_w, y,
                                                                                         y_dtype, V, D, scale);
  ULM_LAUNCH_CHECK("embedding_fwd_kernel");
  return ULM_OK;
}

extern "C" int64_t ulm_embedding_bwd_work_bytes(int64_t N, int64_t V, int64_t D) {
  if (N < 0 || V < 0 || D < 0) return -1;
  return 256;
}

extern "C" int ulm_embedding_bwd(const int64_t* tokens, const void* dy, int dy_dtype, void* dw, int dw_dtype, void* work,
                                 int64_t N, int64_t V, int64_t D, float scale, void* stream) {
  if (int rc = emb_check(tokens, N, V, D)) return rc;
  ULM_REQUIRE(emb_dtype_ok(dy_dtype) && emb_dtype_ok(dw_dtype), "bad dtype");
  ULM_REQUIRE(dw && (N == 0 || (dy && work)), "null pointer argument");
  embedding_bwd_kernel<<<(unsigned)V, EMB_THREADS, 0, static_cast<cudaStream_t>(stream)>>>(tokens, dy, dy_dtype, dw,
                                                                                         dw_dtype, N, D, scale);
  ULM_LAUNCH_CHECK("embedding_bwd_kernel");
  return ULM_OK;
}
