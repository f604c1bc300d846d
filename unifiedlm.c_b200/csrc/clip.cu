// The global 2-norm of many gradient tensors, and clipping by it:
//   n = sqrt(sum over all tensors of g^2),   f = min(1, max_norm / (n + 1e-6)),   out = f g
// One launch per table of tensors adds up the squares, a second one scales. Squares are added in
// fp64 (they do not overflow, and the sum's order does not show in the fp32 norm); each CTA's share of
// the elements is fixed, so the norm has the same bits in every run.
#include <algorithm>
#include <vector>

#include "common.cuh"

namespace ulm {
namespace {

constexpr int CLIP_THREADS = 256;
constexpr int CLIP_CTAS = 592;       // partial sums of one launch
constexpr int CLIP_TABLE = 256;      // tensors of one launch
constexpr int64_t CLIP_CHUNK = 8192; // elements of one piece of work

struct ClipTable {
  const void* in[CLIP_TABLE];
  void* out[CLIP_TABLE];
  int64_t n[CLIP_TABLE];
  int first[CLIP_TABLE];  // index of the tensor's first chunk
  uint8_t in_dtype[CLIP_TABLE], out_dtype[CLIP_TABLE];
  int tensors, chunks;
};

__device__ __forceinline__ int clip_tensor(const ClipTable& t, int chunk) {
  int lo = 0, hi = t.tensors - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.first[mid] <= chunk)
      lo = mid;
    else
      hi = mid - 1;
  }
  return lo;
}

__device__ __forceinline__ float clip_load(const void* p, int dtype, int64_t i) {
  return dtype == ULM_F32 ? static_cast<const float*>(p)[i]
                          : __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}

__device__ __forceinline__ double clip_block_sum(double v, double* red) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
  __syncthreads();
  double s = 0.0;
#pragma unroll
  for (int w = 0; w < CLIP_THREADS / 32; ++w) s += red[w];
  return s;
}

__global__ void __launch_bounds__(CLIP_THREADS)
    grad_square_kernel(const __grid_constant__ ClipTable t, double* __restrict__ part) {
  __shared__ double red[CLIP_THREADS / 32];
  double s = 0.0;
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int j = clip_tensor(t, c);
    const int64_t i0 = (int64_t)(c - t.first[j]) * CLIP_CHUNK, i1 = min(t.n[j], i0 + CLIP_CHUNK);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += CLIP_THREADS) {
      const double g = clip_load(t.in[j], t.in_dtype[j], i);
      s += g * g;
    }
  }
  s = clip_block_sum(s, red);
  if (threadIdx.x == 0) part[blockIdx.x] = s;
}

// the norm from all partial sums, and the clipped gradients
__global__ void __launch_bounds__(CLIP_THREADS)
    grad_clip_kernel(const __grid_constant__ ClipTable t, const double* __restrict__ part, int parts, float max_norm,
                     float* __restrict__ norm, int scale) {
  __shared__ double red[CLIP_THREADS / 32];
  double s = 0.0;
  for (int i = threadIdx.x; i < parts; i += CLIP_THREADS) s += part[i];
  s = clip_block_sum(s, red);
  const float n = (float)sqrt(s);
  if (blockIdx.x == 0 && threadIdx.x == 0) *norm = n;
  if (!scale) return;
  const float q = max_norm / (n + 1e-6f);
  const float f = q > 1.f ? 1.f : q;  // NaN stays
  for (int c = blockIdx.x; c < t.chunks; c += gridDim.x) {
    const int j = clip_tensor(t, c);
    const int64_t i0 = (int64_t)(c - t.first[j]) * CLIP_CHUNK, i1 = min(t.n[j], i0 + CLIP_CHUNK);
    for (int64_t i = i0 + threadIdx.x; i < i1; i += CLIP_THREADS) {
      const float g = clip_load(t.in[j], t.in_dtype[j], i) * f;
      if (t.out_dtype[j] == ULM_F32)
        static_cast<float*>(t.out[j])[i] = g;
      else
        static_cast<__nv_bfloat16*>(t.out[j])[i] = __float2bfloat16_rn(g);
    }
  }
}

// Outputs may not overlap one another, nor a gradient other than their own (which they may be).
int clip_check_overlap(const void* const* grads, void* const* outs, const int64_t* counts, const int* in_dtypes,
                       const int* out_dtypes, int64_t n) {
  struct Range {
    uintptr_t a, b;
    int64_t i;
    bool out;
  };
  std::vector<Range> rs;
  rs.reserve(2 * n);
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    const uintptr_t a = reinterpret_cast<uintptr_t>(grads[i]), o = reinterpret_cast<uintptr_t>(outs[i]);
    rs.push_back({o, o + counts[i] * (out_dtypes[i] == ULM_F32 ? 4 : 2), i, true});
    if (a == o && in_dtypes[i] == out_dtypes[i]) continue;  // in place
    rs.push_back({a, a + counts[i] * (in_dtypes[i] == ULM_F32 ? 4 : 2), i, false});
  }
  std::sort(rs.begin(), rs.end(), [](const Range& x, const Range& y) { return x.a < y.a; });
  uintptr_t end_out = 0, end_any = 0;  // ends of the outputs, and of all ranges, so far
  for (const Range& r : rs) {
    ULM_REQUIRE(!(r.a < end_out || (r.out && r.a < end_any)),
                "gradient %lld overlaps another one's output (the same tensor twice?)", (long long)r.i);
    if (r.out) end_out = std::max(end_out, r.b);
    end_any = std::max(end_any, r.b);
  }
  return ULM_OK;
}

}  // namespace
}  // namespace ulm

using namespace ulm;

extern "C" int64_t ulm_clip_grads_work_bytes(int64_t n) {
  if (n < 0) return -1;
  return std::max<int64_t>(1, cdiv(n, CLIP_TABLE)) * CLIP_CTAS * (int64_t)sizeof(double);
}

static int clip_grads_impl(const void* const* grads, void* const* outs, const int64_t* counts, const int* in_dtypes,
                           const int* out_dtypes, int64_t n, float max_norm, float* norm, void* work, void* stream) {
  ULM_REQUIRE(n >= 0 && n < (1 << 24), "bad number of tensors %lld", (long long)n);
  ULM_REQUIRE(norm && work && (n == 0 || (grads && counts && in_dtypes)), "null pointer argument");
  ULM_REQUIRE(!outs || n == 0 || out_dtypes, "null pointer argument");
  ULM_REQUIRE(!outs || max_norm >= 0.f, "max_norm must not be negative or NaN");
  for (int64_t i = 0; i < n; ++i) {
    ULM_REQUIRE(counts[i] >= 0 && counts[i] < (1ll << 42), "bad element count of tensor %lld", (long long)i);
    ULM_REQUIRE(counts[i] == 0 || (grads[i] && (!outs || outs[i])), "null tensor %lld", (long long)i);
    ULM_REQUIRE(in_dtypes[i] == ULM_F32 || in_dtypes[i] == ULM_BF16, "bad dtype of tensor %lld", (long long)i);
    ULM_REQUIRE(!outs || out_dtypes[i] == ULM_F32 || out_dtypes[i] == ULM_BF16, "bad dtype of tensor %lld", (long long)i);
  }
  if (outs)
    if (int rc = clip_check_overlap(grads, outs, counts, in_dtypes, out_dtypes, n)) return rc;
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  double* part = static_cast<double*>(work);
  std::vector<ClipTable> tables(1);
  tables[0].tensors = tables[0].chunks = 0;
  for (int64_t i = 0; i < n; ++i) {
    if (counts[i] == 0) continue;
    if (tables.back().tensors == CLIP_TABLE) {
      tables.emplace_back();
      tables.back().tensors = tables.back().chunks = 0;
    }
    ClipTable& t = tables.back();
    const int j = t.tensors++;
    t.in[j] = grads[i];
    t.out[j] = outs ? outs[i] : nullptr;
    t.n[j] = counts[i];
    t.in_dtype[j] = (uint8_t)in_dtypes[i];
    t.out_dtype[j] = (uint8_t)(outs ? out_dtypes[i] : 0);
    t.first[j] = t.chunks;
    const int64_t c = t.chunks + cdiv(counts[i], CLIP_CHUNK);
    ULM_REQUIRE(c < (1ll << 31), "too many elements");
    t.chunks = (int)c;
  }
  int parts = 0;
  for (const ClipTable& t : tables) {
    const int ctas = std::max(1, std::min(t.chunks, CLIP_CTAS));
    grad_square_kernel<<<ctas, CLIP_THREADS, 0, st>>>(t, part + parts);
    ULM_LAUNCH_CHECK("grad_square_kernel");
    parts += ctas;
  }
  for (const ClipTable& t : tables) {
    const int ctas = outs ? std::max(1, std::min(t.chunks, CLIP_CTAS)) : 1;
    grad_clip_kernel<<<ctas, CLIP_THREADS, 0, st>>>(t, part, parts, max_norm, norm, outs ? 1 : 0);
    ULM_LAUNCH_CHECK("grad_clip_kernel");
    if (!outs) break;
  }
  return ULM_OK;
}

extern "C" int ulm_clip_grads(const void* const* grads, void* const* outs, const int64_t* counts, const int* in_dtypes,
                              const int* out_dtypes, int64_t n, float max_norm, float* norm, void* work, void* stream) {
  try {
    return clip_grads_impl(grads, outs, counts, in_dtypes, out_dtypes, n, max_norm, norm, work, stream);
  } catch (const std::exception& e) {
    set_error("%s", e.what());
    return ULM_ERR_INVALID;
  }
}
