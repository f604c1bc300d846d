// Token embedding with a scale, and its weight's gradient:
//   y_n = scale * W[t_n],   dW_v = scale * sum over the positions n with t_n = v of dy_n
// Token -1 is padding: a zero row, no gradient. Any other token outside [0, V) gives a NaN row and
// takes no gradient (there is no row to put it in).
//
// Forward: one pass (read N rows, write N rows). 16384 x 768 fp32, which L2 holds: 14 us; bound by HBM beyond:
// 131072 rows of a table of 128000 126 us (5.2 TB/s).
//
// Backward: read dy, write dW, most of whose rows are zero. Three launches:
//   1. embed_sort_kernel: one cluster of 8 CTAs sorts (token, position) by token, stably (radix, 8 bits
//      a pass, counts exchanged over distributed shared memory), while all other CTAs fill dW with
//      zeros (16384 tokens: 13.7 us, about as long as 98 MB of zeros).
//   2. embed_sum_kernel: a warp takes 32 consecutive sorted entries and a block of columns, adds the rows
//      of dy of each run of equal tokens, and writes the runs that lie inside its chunk to dW. A run that
//      crosses chunks (a frequent token: text has a few that make up a tenth of all positions) leaves
//      one partial row a chunk: work is split by positions, not by tokens, so it is even.
//   3. embed_join_kernel: adds the partial rows of the crossing runs.
// Every sum has one fixed order (no float atomics): the same bits in every run. 16384 x 768 fp32 into
// 32000 rows takes 40 us.
#include "common.cuh"

namespace ulm {
namespace {

constexpr int EMB_THREADS = 256;

__device__ __forceinline__ float emb_nan() { return __uint_as_float(0x7FC00000u); }

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

// 16 bytes of E elements as floats and back
template <typename E>
struct EmbVec;
template <>
struct EmbVec<float> {
  static constexpr int N = 4;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[4]) {
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
struct EmbVec<__nv_bfloat16> {
  static constexpr int N = 8;
  static __device__ __forceinline__ void unpack(const uint4& q, float (&x)[8]) {
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

// ---- forward -------------------------------------------------------------------------------------------

// Rows of whole 16-byte pieces, y of W's type: tpr threads a row (a warp for rows of 32 pieces or more),
// four rows a thread so that the look-up of the tokens and the rows' loads overlap.
template <typename E>
__global__ void __launch_bounds__(EMB_THREADS)
    embed_fwd_vec_kernel(const int64_t* __restrict__ tokens, const E* __restrict__ w, int64_t ld_w, E* __restrict__ y,
                         int64_t N, int64_t V, int pieces, int tpr, float scale) {
  pdl_enter();
  constexpr int NV = EmbVec<E>::N, R = 4;
  const int rows = EMB_THREADS / tpr;  // rows of the CTA side by side
  const int64_t n0 = (int64_t)blockIdx.x * rows * R + threadIdx.x / tpr;
  int64_t t[R];
#pragma unroll
  for (int i = 0; i < R; ++i) t[i] = n0 + i * rows < N ? tokens[n0 + i * rows] : -1;
  for (int c = threadIdx.x % tpr; c < pieces; c += tpr) {
    uint4 q[R];
#pragma unroll
    for (int i = 0; i < R; ++i)
      q[i] = t[i] >= 0 && t[i] < V ? reinterpret_cast<const uint4*>(w + t[i] * ld_w)[c] : make_uint4(0, 0, 0, 0);
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (n0 + i * rows >= N) break;
      if (scale != 1.f || t[i] < -1 || t[i] >= V) {
        float x[NV];
        EmbVec<E>::unpack(q[i], x);
#pragma unroll
        for (int j = 0; j < NV; ++j) x[j] = t[i] < -1 || t[i] >= V ? emb_nan() : t[i] == -1 ? 0.f : x[j] * scale;
        q[i] = EmbVec<E>::pack(x);
      }
      reinterpret_cast<uint4*>(y + (n0 + i * rows) * (int64_t)pieces * NV)[c] = q[i];
    }
  }
}

// any strides, widths and types: a warp a row
__global__ void __launch_bounds__(EMB_THREADS)
    embed_fwd_kernel(const int64_t* __restrict__ tokens, const void* __restrict__ w, int w_dtype, int64_t ld_w,
                     void* __restrict__ y, int y_dtype, int64_t N, int64_t V, int64_t D, float scale) {
  pdl_enter();
  const int64_t n = (int64_t)blockIdx.x * (EMB_THREADS / 32) + (threadIdx.x >> 5);
  if (n >= N) return;
  const int64_t t = tokens[n];
#pragma unroll 4
  for (int64_t d = threadIdx.x & 31; d < D; d += 32) {
    float v = t == -1 ? 0.f : emb_nan();
    if (t >= 0 && t < V) v = emb_load(w, w_dtype, t * ld_w + d) * scale;
    emb_store(y, y_dtype, n * D + d, v);
  }
}

// ---- backward: sort ------------------------------------------------------------------------------------

constexpr int SORT_CTAS = 8;  // one cluster
constexpr int SORT_THREADS = 1024;
constexpr int SORT_WARPS = SORT_THREADS / 32;
constexpr int SORT_BINS = 256;
constexpr int SORT_AHEAD = 4;  // entries of a lane loaded before the first is used
constexpr int EMB_FILL_CTAS = 288;  // with the sort's, two CTAs of 1024 threads on each SM

// A shared-memory word of CTA `rank` of the cluster
__device__ __forceinline__ uint32_t ld_cluster_u32(const uint32_t* p, uint32_t rank) {
  uint32_t v;
  asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(mapa_shared(smem_u32(p), rank)) : "memory");
  return v;
}

// Zeroes over `bytes` bytes at p (element size 2 or 4), by threads i, i + n, ...
__device__ __forceinline__ void emb_fill(char* p, int64_t bytes, int64_t i, int64_t n) {
  int64_t head = (16 - (reinterpret_cast<uintptr_t>(p) & 15)) & 15;
  if (head > bytes) head = bytes;
  const int64_t body = (bytes - head) / 16, tail = head + body * 16;
  for (int64_t b = 2 * i; b < head; b += 2 * n) *reinterpret_cast<uint16_t*>(p + b) = 0;
  uint4* v = reinterpret_cast<uint4*>(p + head);
#pragma unroll 4
  for (int64_t b = i; b < body; b += n) v[b] = make_uint4(0, 0, 0, 0);
  for (int64_t b = tail + 2 * i; b < bytes; b += 2 * n) *reinterpret_cast<uint16_t*>(p + b) = 0;
}

// The lanes of the warp that hold the same digit, of those with one (Nine votes: match.any took 8700 cycles
// where they take 5600.)
__device__ __forceinline__ uint32_t sort_same(int digit, bool has) {
  uint32_t same = __ballot_sync(0xffffffffu, has);
#pragma unroll
  for (int b = 0; b < 8; ++b) {
    const bool bit = (digit >> b) & 1;
    const uint32_t set = __ballot_sync(0xffffffffu, bit);
    same &= bit ? set : ~set;
  }
  return same;
}

// CTAs 0 .. 7: the sorted (key, position) pairs, keys the tokens, or V for what is none (these come last).
// Each warp owns a run of consecutive entries. A pass counts digits by warp, turns the counts into the
// warps' first places (over the warps, the CTAs, and the digits), and moves the entries in order, key and
// position in one 8-byte store (the scattered stores bound a pass: 32 sectors a warp). `sorted` holds two
// buffers of N; pass p writes buffer p % 2. All other CTAs zero dW.
__global__ void __cluster_dims__(SORT_CTAS, 1, 1) __launch_bounds__(SORT_THREADS)
    embed_sort_kernel(const int64_t* __restrict__ tokens, int2* __restrict__ sorted, int N, int V,
                      int passes, char* __restrict__ dw, int64_t dw_bytes) {
  __shared__ uint32_t cnt[SORT_WARPS][SORT_BINS];
  __shared__ uint32_t total[SORT_BINS], base[SORT_BINS], wsum[SORT_BINS / 32];
  pdl_enter();
  if (blockIdx.x >= SORT_CTAS) {
    emb_fill(dw, dw_bytes, (int64_t)(blockIdx.x - SORT_CTAS) * SORT_THREADS + threadIdx.x,
             (int64_t)(gridDim.x - SORT_CTAS) * SORT_THREADS);
    return;
  }
  const uint32_t rank = cluster_ctarank();
  const int tid = threadIdx.x, lane = tid & 31, w = tid >> 5;
  const int64_t own = ((int64_t)N + SORT_CTAS * SORT_WARPS * 32 - 1) / (SORT_CTAS * SORT_WARPS * 32) * 32;
  const int64_t i0 = ((int64_t)rank * SORT_WARPS + w) * own, i1 = min((int64_t)N, i0 + own);
  for (int p = 0; p < passes; ++p) {
    const int2* src = sorted + (int64_t)((p + 1) & 1) * N;
    int2* dst = sorted + (int64_t)(p & 1) * N;
    auto load = [&](int64_t i) -> int2 {
      if (i >= i1) return make_int2(-1, 0);
      if (p > 0) return __ldcg(src + i);
      const int64_t t = tokens[i];
      return make_int2(t >= 0 && t < V ? (int)t : V, (int)i);
    };
    for (int b = lane; b < SORT_BINS; b += 32) cnt[w][b] = 0;
    __syncwarp();
    for (int64_t i = i0; i < i1; i += 32 * SORT_AHEAD) {
      int k[SORT_AHEAD];
#pragma unroll
      for (int j = 0; j < SORT_AHEAD; ++j) k[j] = load(i + 32 * j + lane).x;
#pragma unroll
      for (int j = 0; j < SORT_AHEAD; ++j) {
        if (i + 32 * j >= i1) break;
        const int d = (k[j] >> (8 * p)) & (SORT_BINS - 1);
        const uint32_t same = sort_same(d, k[j] >= 0);
        if (k[j] >= 0 && lane == __ffs(same) - 1) cnt[w][d] += __popc(same);
        __syncwarp();
      }
    }
    __syncthreads();
    if (tid < SORT_BINS) {
      uint32_t s = 0;
#pragma unroll 8
      for (int j = 0; j < SORT_WARPS; ++j) {
        const uint32_t c = cnt[j][tid];
        cnt[j][tid] = s;
        s += c;
      }
      total[tid] = s;
    }
    cluster_sync_all();
    uint32_t all = 0, before = 0, incl = 0;
    if (tid < SORT_BINS) {
#pragma unroll
      for (uint32_t c = 0; c < SORT_CTAS; ++c) {
        const uint32_t v = ld_cluster_u32(&total[tid], c);
        all += v;
        if (c < rank) before += v;
      }
      incl = all;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t v = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += v;
      }
      if (lane == 31) wsum[w] = incl;
    }
    __syncthreads();
    if (tid < SORT_BINS) {
      uint32_t off = 0;
      for (int j = 0; j < w; ++j) off += wsum[j];
      base[tid] = off + incl - all + before;
    }
    __syncthreads();
    for (int64_t i = i0; i < i1; i += 32 * SORT_AHEAD) {
      int2 e[SORT_AHEAD];
#pragma unroll
      for (int j = 0; j < SORT_AHEAD; ++j) e[j] = load(i + 32 * j + lane);
#pragma unroll
      for (int j = 0; j < SORT_AHEAD; ++j) {
        if (i + 32 * j >= i1) break;
        const int d = (e[j].x >> (8 * p)) & (SORT_BINS - 1);
        const uint32_t same = sort_same(d, e[j].x >= 0);
        uint32_t to = 0;
        if (e[j].x >= 0) to = base[d] + cnt[w][d] + __popc(same & ((1u << lane) - 1u));
        __syncwarp();
        if (e[j].x >= 0) {
          if (lane == __ffs(same) - 1) cnt[w][d] += __popc(same);
          dst[to] = e[j];
        }
        __syncwarp();
      }
    }
    // the places of this pass are read by the whole cluster in the next one
    cluster_sync_all();
  }
}

// ---- backward: sums ------------------------------------------------------------------------------------

constexpr int EMB_CHUNK = 32;  // sorted entries of one warp

// One warp: entries c * 32 .. of the sorted list, columns d0 .. d0 + 32 NV of D (NV = 1: any alignment).
// part (2 chunks, D) fp32: row 2c the chunk's share of a run that began before it, row 2c + 1 its share
// of a run that begins in it and goes on.
template <typename E, int NV>
__global__ void __launch_bounds__(EMB_THREADS)
    embed_sum_kernel(const int2* __restrict__ sorted, const E* __restrict__ dy,
                     void* __restrict__ dw, int dw_dtype, float* __restrict__ part, int N, int V, int64_t D,
                     int col_blocks, float scale) {
  pdl_enter();
  const int lane = threadIdx.x & 31;
  const int64_t item = (int64_t)blockIdx.x * (EMB_THREADS / 32) + (threadIdx.x >> 5);
  const int64_t c = item / col_blocks;
  const int64_t i0 = c * EMB_CHUNK;
  if (i0 >= N) return;
  const int64_t d = (item - c * col_blocks) * (32 * NV) + lane * NV;
  const bool in = d < D;
  const int n = (int)min((int64_t)EMB_CHUNK, N - i0);
  const int2 mine = lane < n ? sorted[i0 + lane] : make_int2(V, 0);
  const int k = mine.x, p = mine.y;
  const int next_chunk = i0 + EMB_CHUNK < N ? sorted[i0 + EMB_CHUNK].x : V;
  const int last_chunk = i0 > 0 ? sorted[i0 - 1].x : -1;
  int next = __shfl_down_sync(0xffffffffu, k, 1);
  if (lane == EMB_CHUNK - 1) next = next_chunk;
  const uint32_t ends = __ballot_sync(0xffffffffu, k != next);  // entries that end their run
  const uint32_t live = __ballot_sync(0xffffffffu, k < V);
  const bool cont = __shfl_sync(0xffffffffu, k, 0) == last_chunk;
  float acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  bool first = cont;  // the run at hand began before this chunk
  const int m = __popc(live);  // the entries of tokens: they come first
  constexpr int U = 8;  // rows in flight
#pragma unroll 1
  for (int j0 = 0; j0 < m; j0 += U) {
    uint4 q[U];  // 16 bytes, or one element in the first word
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int64_t row = __shfl_sync(0xffffffffu, p, (j0 + u) & 31);
      q[u] = make_uint4(0, 0, 0, 0);
      if (in && j0 + u < m) {
        if (NV == 1)
          q[u].x = __float_as_uint(emb_load(dy, sizeof(E) == 4 ? ULM_F32 : ULM_BF16, row * D + d));
        else
          q[u] = *reinterpret_cast<const uint4*>(dy + row * D + d);
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int j = j0 + u;
      if (j >= m) break;
      if (NV == 1) {
        acc[0] += __uint_as_float(q[u].x);
      } else {
        float x[EmbVec<E>::N];
        EmbVec<E>::unpack(q[u], x);
#pragma unroll
        for (int i = 0; i < NV; ++i) acc[i] += x[i % EmbVec<E>::N];
      }
      const bool end = (ends >> j) & 1u;
      if (!end && j + 1 < EMB_CHUNK) continue;
      const int64_t v = __shfl_sync(0xffffffffu, k, j);
      if (in) {
        if (end && !first) {  // the whole run is here
          if (NV == 1) {
            emb_store(dw, dw_dtype, v * D + d, acc[0] * scale);
          } else {
#pragma unroll
            for (int i = 0; i < NV; ++i) acc[i] *= scale;
            if (dw_dtype == ULM_F32) {
#pragma unroll
              for (int i = 0; i + 3 < NV; i += 4)
                reinterpret_cast<uint4*>(static_cast<float*>(dw) + v * D + d)[i / 4] = EmbVec<float>::pack(acc + i);
            } else if (NV == 8) {
              *reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(dw) + v * D + d) =
                  EmbVec<__nv_bfloat16>::pack(acc);
            } else {
#pragma unroll
              for (int i = 0; i < NV; ++i) emb_store(dw, dw_dtype, v * D + d + i, acc[i]);
            }
          }
        } else {
          float* o = part + (2 * c + (first ? 0 : 1)) * D + d;
          if (NV == 1) {
            o[0] = acc[0];
          } else {
#pragma unroll
            for (int i = 0; i + 3 < NV; i += 4) reinterpret_cast<uint4*>(o)[i / 4] = EmbVec<float>::pack(acc + i);
          }
        }
      }
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] = 0.f;
      first = false;
    }
  }
}

// CTA (c, block of 32 NV columns): if a run begins in chunk c and goes on, the sum of its shares: warp w
// adds every eighth one, then the warps' sums are added in order.
template <int NV>
__global__ void __launch_bounds__(EMB_THREADS)
    embed_join_kernel(const int2* __restrict__ sorted, const float* __restrict__ part, void* __restrict__ dw, int dw_dtype,
                      int N, int V, int64_t D, float scale) {
  pdl_enter();
  __shared__ float red[EMB_THREADS / 32][32 * NV];
  const int lane = threadIdx.x & 31, w = threadIdx.x >> 5;
  const int64_t c = blockIdx.x, i0 = c * EMB_CHUNK, last = i0 + EMB_CHUNK - 1;
  if (last + 1 >= N) return;
  const int k = sorted[last].x, after = sorted[last + 1].x, begin = sorted[i0].x;
  const int before = i0 > 0 ? sorted[i0 - 1].x : -1;
  if (k >= V || after != k) return;            // no run goes on
  if (begin == k && before == k) return;       // it began in an earlier chunk
  // chunks c + 1 .. c + more begin with entries of the same run
  const int64_t chunks = (N + EMB_CHUNK - 1) / EMB_CHUNK;
  int64_t more = 0;
  for (;;) {
    const int64_t cc = c + 1 + more + lane;
    const uint32_t b = __ballot_sync(0xffffffffu, cc < chunks && sorted[cc * EMB_CHUNK].x == k);
    if (b == 0xffffffffu) {
      more += 32;
    } else {
      more += __ffs(~b) - 1;
      break;
    }
  }
  const int64_t d = ((int64_t)blockIdx.y * 32 + lane) * NV;
  float acc[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) acc[i] = 0.f;
  if (d < D) {
#pragma unroll 8
    for (int64_t j = w; j <= more; j += EMB_THREADS / 32) {
      const float* p = part + (j == 0 ? 2 * c + 1 : 2 * (c + j)) * D + d;
      float x[NV];
      if (NV == 4)
        *reinterpret_cast<float4*>(x) = *reinterpret_cast<const float4*>(p);
      else
        x[0] = p[0];
#pragma unroll
      for (int i = 0; i < NV; ++i) acc[i] += x[i];
    }
  }
#pragma unroll
  for (int i = 0; i < NV; ++i) red[w][lane + 32 * i] = acc[i];
  __syncthreads();
  if (w == 0 && d < D) {
#pragma unroll
    for (int i = 0; i < NV; ++i) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < EMB_THREADS / 32; ++j) s += red[j][lane + 32 * i];
      emb_store(dw, dw_dtype, (int64_t)k * D + d + i, s * scale);
    }
  }
}

int emb_check(const int64_t* tokens, int64_t N, int64_t V, int64_t D) {
  ULM_REQUIRE(N >= 0 && V > 0 && D > 0, "bad extents N=%lld V=%lld D=%lld", (long long)N, (long long)V, (long long)D);
  ULM_REQUIRE(N < (1ll << 30) && V < (1ll << 30) && D < (1 << 20), "extent too large");
  ULM_REQUIRE(N == 0 || tokens, "null tokens");
  return ULM_OK;
}
bool emb_dtype_ok(int dt) { return dt == ULM_F32 || dt == ULM_BF16; }

struct EmbWork {
  int2* sorted;
  float* part;
  int64_t bytes;
};
EmbWork emb_work(void* base, int64_t N, int64_t D) {
  auto al = [](int64_t n) { return (n + 255) / 256 * 256; };
  char* p = static_cast<char*>(base);
  EmbWork w;
  w.sorted = reinterpret_cast<int2*>(p);
  w.part = reinterpret_cast<float*>(p + al(2 * N * 8));
  w.bytes = al(2 * N * 8) + al(2 * cdiv(N, EMB_CHUNK) * D * 4);
  return w;
}

template <typename E>
int emb_sums(const EmbWork& w, const int2* sorted, const void* dy, void* dw, int dw_dtype, int64_t N,
             int64_t V, int64_t D, float scale, cudaStream_t st) {
  constexpr int NV = EmbVec<E>::N;
  const bool vec = D % 8 == 0 && is_aligned16(dy) && is_aligned16(dw);
  const int64_t cols = cdiv(D, vec ? 32 * NV : 32), chunks = cdiv(N, EMB_CHUNK);
  const int64_t ctas = cdiv(chunks * cols, EMB_THREADS / 32);
  ULM_REQUIRE(ctas < (1ll << 31) && cdiv(D, 32) < 65536, "extent too large");
  auto kern = vec ? embed_sum_kernel<E, NV> : embed_sum_kernel<E, 1>;
  if (int rc = launch_pdl(kern, dim3((unsigned)ctas), dim3(EMB_THREADS), 0, st, sorted, static_cast<const E*>(dy), dw,
                          dw_dtype, w.part, (int)N, (int)V, D, (int)cols, scale))
    return rc;
  if (chunks < 2) return ULM_OK;
  return launch_pdl(vec ? embed_join_kernel<4> : embed_join_kernel<1>,
                    dim3((unsigned)(chunks - 1), (unsigned)cdiv(D, vec ? 128 : 32)), dim3(EMB_THREADS), 0, st, sorted,
                    static_cast<const float*>(w.part), dw, dw_dtype, (int)N, (int)V, D, scale);
}

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
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int nv = w_dtype == ULM_F32 ? 4 : 8;
  if (w_dtype == y_dtype && D % nv == 0 && ld_w % nv == 0 && is_aligned16(weight) && is_aligned16(y)) {
    const int pieces = (int)(D / nv);
    int tpr = 1;
    while (tpr < pieces && tpr < 32) tpr *= 2;
    const dim3 grid((unsigned)cdiv(N, 4 * (EMB_THREADS / tpr)));
    return w_dtype == ULM_F32
               ? launch_pdl(embed_fwd_vec_kernel<float>, grid, dim3(EMB_THREADS), 0, st, tokens,
                            static_cast<const float*>(weight), ld_w, static_cast<float*>(y), N, V, pieces, tpr, scale)
               : launch_pdl(embed_fwd_vec_kernel<__nv_bfloat16>, grid, dim3(EMB_THREADS), 0, st, tokens,
                            static_cast<const __nv_bfloat16*>(weight), ld_w, static_cast<__nv_bfloat16*>(y), N, V, pieces,
                            tpr, scale);
  }
  return launch_pdl(embed_fwd_kernel, dim3((unsigned)cdiv(N, EMB_THREADS / 32)), dim3(EMB_THREADS), 0, st, tokens, weight,
                    w_dtype, ld_w, y, y_dtype, N, V, D, scale);
}

extern "C" int64_t ulm_embedding_bwd_work_bytes(int64_t N, int64_t V, int64_t D) {
  if (N < 0 || V < 0 || D < 0) return -1;
  return emb_work(nullptr, N, D).bytes + 256;
}

extern "C" int ulm_embedding_bwd(const int64_t* tokens, const void* dy, int dy_dtype, void* dw, int dw_dtype, void* work,
                                 int64_t N, int64_t V, int64_t D, float scale, void* stream) {
  if (int rc = emb_check(tokens, N, V, D)) return rc;
  ULM_REQUIRE(emb_dtype_ok(dy_dtype) && emb_dtype_ok(dw_dtype), "bad dtype");
  ULM_REQUIRE(dw && (N == 0 || (dy && work)), "null pointer argument");
  cudaStream_t st = static_cast<cudaStream_t>(stream);
  const int64_t dw_bytes = V * D * (dw_dtype == ULM_F32 ? 4 : 2);
  if (N == 0) {
    ULM_CUDA_TRY(cudaMemsetAsync(dw, 0, dw_bytes, st));
    return ULM_OK;
  }
  ULM_REQUIRE(is_aligned16(work), "work must be 16-byte aligned");
  const EmbWork w = emb_work(work, N, D);
  int passes = 1;
  while (V >> (8 * passes)) ++passes;  // keys are 0 .. V
  if (int rc = launch_pdl(embed_sort_kernel, dim3(SORT_CTAS + EMB_FILL_CTAS), dim3(SORT_THREADS), 0, st, tokens,
                          w.sorted, (int)N, (int)V, passes, static_cast<char*>(dw), dw_bytes))
    return rc;
  const int64_t last = (int64_t)((passes - 1) & 1) * N;
  return dy_dtype == ULM_F32 ? emb_sums<float>(w, w.sorted + last, dy, dw, dw_dtype, N, V, D, scale, st)
                             : emb_sums<__nv_bfloat16>(w, w.sorted + last, dy, dw, dw_dtype, N, V, D, scale, st);
}
