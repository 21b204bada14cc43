// The token side of a MoE layer, each step with its gradient: the experts of every token and their weights (route), the
// tokens copied into the order of their experts (permute) and the weighted sum of a token's rows (unpermute). All of it
// is bound by memory; every sum is in fp32 and in a fixed order, so results do not change from run to run.
//
// `scatter_index` [ntokens, topk] holds the row of every (token, choice) pair, as fluxb_moe_scatter_index makes it: the
// valid entries are the rows 0 .. sum(splits) - 1, each once; an entry outside [0, ntokens * topk) is a pair without an
// expert and takes no part. The rows from sum(splits) on belong to nobody: what is written there is zero.
#include "internal.h"

namespace fluxb {

// ----------------------------------------------------------------------------------------------------------- route
// z: logits of a token. chosen = the topk largest (ties: the lower expert), w = softmax over the chosen ones:
//   w_j = exp(z_j - z_max) / sum_i exp(z_i - z_max),   dz_j = w_j (dw_j - sum_i w_i dw_i),   0 for the others.
// One warp per token, its logits in registers as order-preserving integers; a choice is two warp-wide integer
// reductions (the largest key, the lowest expert that has it), and only the lane that held it looks for its next one.
constexpr int kRouteThreads = 128;
constexpr int kRouteMaxExperts = 1024;
constexpr int kRouteMaxTopk = 32;

template <class T>
__device__ __forceinline__ float to_f32(T v);
template <>
__device__ __forceinline__ float to_f32(float v) { return v; }
template <>
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
template <>
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v);
template <>
__device__ __forceinline__ float from_f32(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f32(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half from_f32(float v) { return __float2half_rn(v); }

// Integers in the order of the floats: 0 = not to be chosen (minus infinity), NaN above all.
__device__ __forceinline__ uint32_t route_key(float v) {
  if (v != v) return 0xFFFFFFFFu;
  if (v == -INFINITY) return 0u;
  const uint32_t u = __float_as_uint(v + 0.0f);  // -0 equals +0
  return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float route_value(uint32_t key) {
  if (key == 0xFFFFFFFFu) return __uint_as_float(0x7FC00000u);
  return __uint_as_float((key & 0x80000000u) ? key ^ 0x80000000u : ~key);
}

template <class T, int VPL>
__global__ void __launch_bounds__(kRouteThreads)
moe_route_kernel(const T* __restrict__ logits, int ntokens, int nexperts, int topk, int* __restrict__ chosen, float* __restrict__ weights) {
  const int lane = threadIdx.x & 31;
  const int t = static_cast<int>((static_cast<long long>(blockIdx.x) * kRouteThreads + threadIdx.x) >> 5);
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (t >= ntokens) return;
  const T* z = logits + static_cast<long long>(t) * nexperts;
  uint32_t key[VPL];
#pragma unroll
  for (int i = 0; i < VPL; ++i) key[i] = lane + 32 * i < nexperts ? route_key(to_f32(z[lane + 32 * i])) : 0u;
  uint32_t best = 0;
  int at = 0;
  auto look = [&] {
    best = 0;
    at = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (key[i] > best) {
        best = key[i];
        at = i;
      }
  };
  look();
  int mine = -1;         // lane j: choice j
  uint32_t mine_key = 0;
  for (int j = 0; j < topk; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    if (top == 0u) break;  // nothing left that may be chosen
    const unsigned e = __reduce_min_sync(0xffffffffu, best == top ? static_cast<unsigned>(lane + 32 * at) : 0x7FFFFFFFu);
    if (lane == j) {
      mine = static_cast<int>(e);
      mine_key = top;
    }
    if (static_cast<int>(e & 31u) == lane) {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (static_cast<int>(e >> 5) == i) key[i] = 0u;
      look();
    }
  }
  const float v = route_value(mine_key);
  const float top_v = __shfl_sync(0xffffffffu, v, 0);
  const float p = mine >= 0 ? expf(v - top_v) : 0.0f;
  float sum = p;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (lane < topk) {
    const long long o = static_cast<long long>(t) * topk + lane;
    chosen[o] = mine;
    weights[o] = mine >= 0 ? p / sum : 0.0f;
  }
}

template <class T>
__global__ void __launch_bounds__(kRouteThreads)
moe_route_backward_kernel(const float* __restrict__ dweights, const int* __restrict__ chosen, const float* __restrict__ weights,
                          int ntokens, int nexperts, int topk, T* __restrict__ dlogits) {
  const int lane = threadIdx.x & 31;
  const int t = static_cast<int>((static_cast<long long>(blockIdx.x) * kRouteThreads + threadIdx.x) >> 5);
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (t >= ntokens) return;
  int c = -1;
  float w = 0.0f, dw = 0.0f;
  if (lane < topk) {
    const long long o = static_cast<long long>(t) * topk + lane;
    c = chosen[o];
    if (c >= 0) {
      w = weights[o];
      dw = dweights[o];
    }
  }
  float s = w * dw;
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  const float g = w * (dw - s);
  T* out = dlogits + static_cast<long long>(t) * nexperts;
  for (int e0 = 0; e0 < nexperts; e0 += 32) {
    float v = 0.0f;
    for (int j = 0; j < topk; ++j) {
      const int cj = __shfl_sync(0xffffffffu, c, j);
      const float gj = __shfl_sync(0xffffffffu, g, j);
      if (cj == e0 + lane) v = gj;
    }
    if (e0 + lane < nexperts) out[e0 + lane] = from_f32<T>(v);
  }
}

// ---------------------------------------------------------------------------------------------------- permute, unpermute
constexpr int kSortThreads = 256;
constexpr int kSortTailCtas = 148;  // the rows that belong to nobody are cleared by CTAs of their own

template <int VB>
struct RawVec;
template <>
struct RawVec<16> { using type = uint4; };
template <>
struct RawVec<8> { using type = uint2; };
template <>
struct RawVec<4> { using type = uint32_t; };
template <>
struct RawVec<2> { using type = uint16_t; };
template <>
struct RawVec<1> { using type = uint8_t; };

template <class T, int VB>
struct SortVec {
  static constexpr int N = VB / static_cast<int>(sizeof(T));
  union {
    typename RawVec<VB>::type raw;
    T e[N];
  };
  __device__ __forceinline__ SortVec() {}
};

// rows [sum(splits), rows) of a matrix with `row_vecs` vectors a row are cleared by the CTAs tail_cta of tail_ctas
template <int VB>
__device__ __forceinline__ void sort_clear_tail(typename RawVec<VB>::type* rows_out, long long rows, long long row_vecs, const int* splits,
                                                int nexperts, int tail_cta, int tail_ctas) {
  __shared__ long long part[kSortThreads / 32];
  long long s = 0;
  for (int e = threadIdx.x; e < nexperts; e += kSortThreads) s += splits[e];
#pragma unroll
  for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
  __syncthreads();
  s = 0;
#pragma unroll
  for (int w = 0; w < kSortThreads / 32; ++w) s += part[w];
  if (s < 0) s = 0;
  typename RawVec<VB>::type zero;
  memset(&zero, 0, sizeof(zero));
  for (long long r = s + tail_cta; r < rows; r += tail_ctas)
    for (long long v = threadIdx.x; v < row_vecs; v += kSortThreads) rows_out[r * row_vecs + v] = zero;
}

// `width` threads (a power of two from 32 to 256) take one token: each vector is read once and stored to the token's rows.
template <int VB>
__global__ void __launch_bounds__(kSortThreads)
moe_permute_kernel(const typename RawVec<VB>::type* __restrict__ tokens, int ntokens, int topk, int row_vecs, int width, int main_ctas,
                   const int* __restrict__ splits, int nexperts, const int* __restrict__ index,
                   typename RawVec<VB>::type* __restrict__ rows_out) {
  const long long rows = static_cast<long long>(ntokens) * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (static_cast<int>(blockIdx.x) >= main_ctas) {
    sort_clear_tail<VB>(rows_out, rows, row_vecs, splits, nexperts, static_cast<int>(blockIdx.x) - main_ctas, static_cast<int>(gridDim.x) - main_ctas);
    return;
  }
  const int per = kSortThreads / width;
  const long long t = static_cast<long long>(blockIdx.x) * per + static_cast<int>(threadIdx.x) / width;
  if (t >= ntokens) return;
  const auto* src = tokens + t * row_vecs;
  const int* idx = index + t * topk;
  constexpr int UN = 4;
  for (int v0 = static_cast<int>(threadIdx.x) & (width - 1); v0 < row_vecs; v0 += UN * width) {
    typename RawVec<VB>::type x[UN];
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (v0 + u * width < row_vecs) x[u] = __ldg(src + v0 + u * width);
    for (int j = 0; j < topk; ++j) {
      const int r = idx[j];
      if (r < 0 || r >= rows) continue;
      auto* dst = rows_out + static_cast<long long>(r) * row_vecs;
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (v0 + u * width < row_vecs) dst[v0 + u * width] = x[u];
    }
  }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, long long i) {
  if (dtype == FLUXB_F32) return static_cast<const float*>(w)[i];
  if (dtype == FLUXB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// out[t] = sum_j w[t, j] rows[index[t, j]], j ascending, rounded once; without weights the plain sum
template <class T, int VB>
__global__ void __launch_bounds__(kSortThreads)
moe_unpermute_kernel(const typename RawVec<VB>::type* __restrict__ rows_in, int ntokens, int topk, int row_vecs, int width,
                     const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                     typename RawVec<VB>::type* __restrict__ out) {
  using V = SortVec<T, VB>;
  const long long rows = static_cast<long long>(ntokens) * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const int per = kSortThreads / width;
  const long long t = static_cast<long long>(blockIdx.x) * per + static_cast<int>(threadIdx.x) / width;
  if (t >= ntokens) return;
  const int* idx = index + t * topk;
  constexpr int UN = 4;  // rows whose loads are in flight together
  for (int v = static_cast<int>(threadIdx.x) & (width - 1); v < row_vecs; v += width) {
    float acc[V::N];
#pragma unroll
    for (int i = 0; i < V::N; ++i) acc[i] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += UN) {
      V x[UN];
      float w[UN];
      bool ok[UN];
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        const int r = j0 + u < topk ? idx[j0 + u] : -1;
        ok[u] = r >= 0 && r < rows;
        w[u] = 1.0f;
        if (ok[u]) {
          x[u].raw = __ldg(rows_in + static_cast<long long>(r) * row_vecs + v);
          if (weights != nullptr) w[u] = load_weight(weights, wdtype, t * topk + j0 + u);
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (ok[u]) {
#pragma unroll
          for (int i = 0; i < V::N; ++i) acc[i] = fmaf(w[u], to_f32(x[u].e[i]), acc[i]);
        }
    }
    V y;
#pragma unroll
    for (int i = 0; i < V::N; ++i) y.e[i] = from_f32<T>(acc[i]);
    out[t * row_vecs + v] = y.raw;
  }
}

// drows[index[t, j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], rows[index[t, j]]>, KC choices at a time: dout is read
// once for them, their rows' loads are in flight together, and the products stay in fp32 until the token's threads add
// them up. `rows_in` and `dweights` are null where only drows is wanted.
template <class T, int VB, int KC>
__global__ void __launch_bounds__(kSortThreads)
moe_unpermute_backward_kernel(const typename RawVec<VB>::type* __restrict__ dout, const typename RawVec<VB>::type* __restrict__ rows_in,
                              int ntokens, int topk, int row_vecs, int width, int main_ctas, const int* __restrict__ splits, int nexperts,
                              const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                              typename RawVec<VB>::type* __restrict__ drows, void* __restrict__ dweights) {
  using V = SortVec<T, VB>;
  __shared__ float part[kSortThreads / 32][KC];
  const long long rows = static_cast<long long>(ntokens) * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (static_cast<int>(blockIdx.x) >= main_ctas) {
    if (drows != nullptr)
      sort_clear_tail<VB>(drows, rows, row_vecs, splits, nexperts, static_cast<int>(blockIdx.x) - main_ctas, static_cast<int>(gridDim.x) - main_ctas);
    return;
  }
  const int per = kSortThreads / width;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const long long t = static_cast<long long>(blockIdx.x) * per + tid / width;
  const bool live = t < ntokens;  // (all threads of the CTA meet at the barriers)
  for (int j0 = 0; j0 < topk; j0 += KC) {
    int row[KC];
    float w[KC], dot[KC];
#pragma unroll
    for (int u = 0; u < KC; ++u) {
      int r = live && j0 + u < topk ? index[t * topk + j0 + u] : -1;
      if (r >= rows) r = -1;
      row[u] = r;
      w[u] = r >= 0 ? load_weight(weights, wdtype, t * topk + j0 + u) : 0.0f;
      dot[u] = 0.0f;
    }
    if (live) {
      for (int v = tid & (width - 1); v < row_vecs; v += width) {
        V g, x[KC];
        g.raw = __ldg(dout + t * row_vecs + v);
        if (rows_in != nullptr) {
#pragma unroll
          for (int u = 0; u < KC; ++u)
            if (row[u] >= 0) x[u].raw = __ldg(rows_in + static_cast<long long>(row[u]) * row_vecs + v);
        }
#pragma unroll
        for (int u = 0; u < KC; ++u) {
          if (row[u] < 0) continue;
          if (rows_in != nullptr) {
#pragma unroll
            for (int i = 0; i < V::N; ++i) dot[u] = fmaf(to_f32(g.e[i]), to_f32(x[u].e[i]), dot[u]);
          }
          if (drows != nullptr) {
            V d;
#pragma unroll
            for (int i = 0; i < V::N; ++i) d.e[i] = from_f32<T>(w[u] * to_f32(g.e[i]));
            drows[static_cast<long long>(row[u]) * row_vecs + v] = d.raw;
          }
        }
      }
    }
    if (dweights == nullptr) continue;
#pragma unroll
    for (int u = 0; u < KC; ++u) {
#pragma unroll
      for (int off = 16; off > 0; off >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], off);
      if (lane == 0) part[warp][u] = dot[u];
    }
    __syncthreads();
    const int u = tid & (width - 1);
    if (live && u < KC && j0 + u < topk) {
      float s = 0.0f;
      for (int k = 0; k < width / 32; ++k) s += part[tid / width * (width / 32) + k][u];
      const long long o = t * topk + j0 + u;
      if (wdtype == FLUXB_F32) static_cast<float*>(dweights)[o] = s;
      else if (wdtype == FLUXB_BF16) static_cast<__nv_bfloat16*>(dweights)[o] = __float2bfloat16_rn(s);
      else static_cast<__half*>(dweights)[o] = __float2half_rn(s);
    }
    __syncthreads();
  }
}

// Widest vector, up to 16 bytes and not below `least`, that divides a row and every pointer.
static int sort_vec_bytes(long long row_bytes, int least, std::initializer_list<const void*> ptrs) {
  uintptr_t a = static_cast<uintptr_t>(row_bytes);
  for (const void* p : ptrs) a |= reinterpret_cast<uintptr_t>(p);
  int vb = 16;
  while (vb > least && (a & static_cast<uintptr_t>(vb - 1)) != 0) vb >>= 1;
  return vb;
}
static int sort_width(long long row_vecs) {
  int w = 32;
  while (w < kSortThreads && w < row_vecs) w *= 2;
  return w;
}

static int check_sort(const char* what, int ntokens, int topk, int hidden) {
  FLUXB_REQUIRE(ntokens >= 0 && topk >= 1 && hidden >= 1 && hidden < (1 << 28), "%s: ntokens=%d topk=%d hidden=%d invalid", what, ntokens, topk, hidden);
  FLUXB_REQUIRE(static_cast<long long>(ntokens) * topk < (1ll << 30), "%s: too many routed rows", what);
  return FLUXB_OK;
}
static bool is_float_type(int dt) { return dt == FLUXB_F32 || dt == FLUXB_BF16 || dt == FLUXB_F16; }

template <class T>
static int launch_route(const void* logits, int ntokens, int nexperts, int topk, int* chosen, float* weights, cudaStream_t stream) {
  const int grid = static_cast<int>((static_cast<long long>(ntokens) * 32 + kRouteThreads - 1) / kRouteThreads);
  const T* z = static_cast<const T*>(logits);
#define FLUXB_ROUTE(V) \
  if (nexperts <= 32 * V) return launch_pdl(moe_route_kernel<T, V>, grid, kRouteThreads, stream, z, ntokens, nexperts, topk, chosen, weights)
  FLUXB_ROUTE(1);
  FLUXB_ROUTE(2);
  FLUXB_ROUTE(4);
  FLUXB_ROUTE(8);
  FLUXB_ROUTE(16);
  FLUXB_ROUTE(32);
#undef FLUXB_ROUTE
  FLUXB_FAIL(FLUXB_ERR_INVALID, "moe_route: nexperts=%d above %d", nexperts, kRouteMaxExperts);
}

template <class T, int VB>
static int launch_unpermute(const void* rows, int ntokens, int topk, int row_vecs, const int* index, const void* weights, int wdtype, void* out,
                            cudaStream_t stream) {
  using R = typename RawVec<VB>::type;
  const int width = sort_width(row_vecs), per = kSortThreads / width;
  return launch_pdl(moe_unpermute_kernel<T, VB>, (ntokens + per - 1) / per, kSortThreads, stream, static_cast<const R*>(rows), ntokens, topk, row_vecs,
                    width, index, weights, wdtype, static_cast<R*>(out));
}

template <class T, int VB>
static int launch_unpermute_backward(const void* dout, const void* rows, int ntokens, int topk, int row_vecs, const int* splits, int nexperts,
                                     const int* index, const void* weights, int wdtype, void* drows, void* dweights, cudaStream_t stream) {
  using R = typename RawVec<VB>::type;
  const int width = sort_width(row_vecs), per = kSortThreads / width;
  const int main_ctas = (ntokens + per - 1) / per;
  const long long total = static_cast<long long>(ntokens) * topk;
  const int tail = total < kSortTailCtas ? static_cast<int>(total) : kSortTailCtas;
  const int grid = main_ctas + (drows != nullptr ? tail : 0);
#define FLUXB_UNPERMUTE_BWD(KC)                                                                                                                    \
  return launch_pdl(moe_unpermute_backward_kernel<T, VB, KC>, grid, kSortThreads, stream, static_cast<const R*>(dout), static_cast<const R*>(rows), \
                    ntokens, topk, row_vecs, width, main_ctas, splits, nexperts, index, weights, wdtype, static_cast<R*>(drows), dweights)
  if (topk <= 2) FLUXB_UNPERMUTE_BWD(2);
  if (topk <= 4) FLUXB_UNPERMUTE_BWD(4);
  FLUXB_UNPERMUTE_BWD(8);
#undef FLUXB_UNPERMUTE_BWD
}

}  // namespace fluxb

using namespace fluxb;

extern "C" {

int fluxb_moe_route(const void* logits, int dtype, int ntokens, int nexperts, int topk, int* chosen_out, float* weights_out,
                    fluxb_stream_t stream) {
  FLUXB_REQUIRE(is_float_type(dtype), "moe_route: logits must be fp32, bf16 or fp16");
  FLUXB_REQUIRE(nexperts >= 1 && nexperts <= kRouteMaxExperts, "moe_route: nexperts=%d out of [1,%d]", nexperts, kRouteMaxExperts);
  FLUXB_REQUIRE(topk >= 1 && topk <= kRouteMaxTopk && topk <= nexperts, "moe_route: topk=%d out of [1,%d] for %d experts", topk, kRouteMaxTopk, nexperts);
  int rc = check_sort("moe_route", ntokens, topk, 1);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(logits != nullptr && chosen_out != nullptr && weights_out != nullptr, "moe_route: NULL argument");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FLUXB_F32) return launch_route<float>(logits, ntokens, nexperts, topk, chosen_out, weights_out, s);
  if (dtype == FLUXB_BF16) return launch_route<__nv_bfloat16>(logits, ntokens, nexperts, topk, chosen_out, weights_out, s);
  return launch_route<__half>(logits, ntokens, nexperts, topk, chosen_out, weights_out, s);
}

int fluxb_moe_route_backward(const float* dweights, const int* chosen, const float* weights, int dtype, int ntokens, int nexperts, int topk,
                             void* dlogits, fluxb_stream_t stream) {
  FLUXB_REQUIRE(is_float_type(dtype), "moe_route_backward: logits must be fp32, bf16 or fp16");
  FLUXB_REQUIRE(nexperts >= 1 && nexperts <= kRouteMaxExperts, "moe_route_backward: nexperts=%d out of [1,%d]", nexperts, kRouteMaxExperts);
  FLUXB_REQUIRE(topk >= 1 && topk <= kRouteMaxTopk && topk <= nexperts, "moe_route_backward: topk=%d out of [1,%d] for %d experts", topk, kRouteMaxTopk,
                nexperts);
  int rc = check_sort("moe_route_backward", ntokens, topk, 1);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(dweights != nullptr && chosen != nullptr && weights != nullptr && dlogits != nullptr, "moe_route_backward: NULL argument");
  const int grid = static_cast<int>((static_cast<long long>(ntokens) * 32 + kRouteThreads - 1) / kRouteThreads);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FLUXB_F32)
    return launch_pdl(moe_route_backward_kernel<float>, grid, kRouteThreads, s, dweights, chosen, weights, ntokens, nexperts, topk, static_cast<float*>(dlogits));
  if (dtype == FLUXB_BF16)
    return launch_pdl(moe_route_backward_kernel<__nv_bfloat16>, grid, kRouteThreads, s, dweights, chosen, weights, ntokens, nexperts, topk,
                      static_cast<__nv_bfloat16*>(dlogits));
  return launch_pdl(moe_route_backward_kernel<__half>, grid, kRouteThreads, s, dweights, chosen, weights, ntokens, nexperts, topk, static_cast<__half*>(dlogits));
}

int fluxb_moe_permute(const void* tokens, int ntokens, int topk, long long row_bytes, const int* splits, int nexperts, const int* scatter_index,
                      void* rows_out, fluxb_stream_t stream) {
  FLUXB_REQUIRE(row_bytes >= 1 && row_bytes < (1ll << 30), "moe_permute: row_bytes=%lld invalid", row_bytes);
  FLUXB_REQUIRE(nexperts >= 1, "moe_permute: nexperts=%d invalid", nexperts);
  int rc = check_sort("moe_permute", ntokens, topk, 1);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(tokens != nullptr && splits != nullptr && scatter_index != nullptr && rows_out != nullptr, "moe_permute: NULL argument");
  const int vb = sort_vec_bytes(row_bytes, 1, {tokens, rows_out});
  const long long row_vecs = row_bytes / vb;
  const int width = sort_width(row_vecs), per = kSortThreads / width;
  const int main_ctas = (ntokens + per - 1) / per;
  const long long total = static_cast<long long>(ntokens) * topk;
  const int grid = main_ctas + (total < kSortTailCtas ? static_cast<int>(total) : kSortTailCtas);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLUXB_PERMUTE(VB)                                                                                                                       \
  return launch_pdl(moe_permute_kernel<VB>, grid, kSortThreads, s, static_cast<const RawVec<VB>::type*>(tokens), ntokens, topk,                  \
                    static_cast<int>(row_vecs), width, main_ctas, splits, nexperts, scatter_index, static_cast<RawVec<VB>::type*>(rows_out))
  switch (vb) {
    case 16: FLUXB_PERMUTE(16);
    case 8: FLUXB_PERMUTE(8);
    case 4: FLUXB_PERMUTE(4);
    case 2: FLUXB_PERMUTE(2);
    default: FLUXB_PERMUTE(1);
  }
#undef FLUXB_PERMUTE
}

#define FLUXB_SORT_TYPES(CALL)                                          \
  do {                                                                  \
    if (dtype == FLUXB_F32) {                                           \
      if (vb == 16) return CALL(float, 16);                             \
      if (vb == 8) return CALL(float, 8);                               \
      return CALL(float, 4);                                            \
    }                                                                   \
    if (dtype == FLUXB_BF16) {                                          \
      if (vb == 16) return CALL(__nv_bfloat16, 16);                     \
      if (vb == 8) return CALL(__nv_bfloat16, 8);                       \
      if (vb == 4) return CALL(__nv_bfloat16, 4);                       \
      return CALL(__nv_bfloat16, 2);                                    \
    }                                                                   \
    if (vb == 16) return CALL(__half, 16);                              \
    if (vb == 8) return CALL(__half, 8);                                \
    if (vb == 4) return CALL(__half, 4);                                \
    return CALL(__half, 2);                                             \
  } while (0)

int fluxb_moe_unpermute(const void* rows, int dtype, int ntokens, int topk, int hidden, const int* scatter_index, const void* weights,
                        int weights_dtype, void* out, fluxb_stream_t stream) {
  FLUXB_REQUIRE(is_float_type(dtype), "moe_unpermute: rows must be fp32, bf16 or fp16");
  FLUXB_REQUIRE(weights == nullptr || is_float_type(weights_dtype), "moe_unpermute: weights must be fp32, bf16 or fp16");
  int rc = check_sort("moe_unpermute", ntokens, topk, hidden);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(rows != nullptr && scatter_index != nullptr && out != nullptr, "moe_unpermute: NULL argument");
  const int eb = dtype_bytes(dtype);
  const long long row_bytes = static_cast<long long>(hidden) * eb;
  const int vb = sort_vec_bytes(row_bytes, eb, {rows, out});
  const int row_vecs = static_cast<int>(row_bytes / vb);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLUXB_CALL(T, VB) launch_unpermute<T, VB>(rows, ntokens, topk, row_vecs, scatter_index, weights, weights_dtype, out, s)
  FLUXB_SORT_TYPES(FLUXB_CALL);
#undef FLUXB_CALL
}

int fluxb_moe_unpermute_backward(const void* dout, const void* rows, int dtype, int ntokens, int topk, int hidden, const int* splits, int nexperts,
                                 const int* scatter_index, const void* weights, int weights_dtype, void* drows, void* dweights,
                                 fluxb_stream_t stream) {
  FLUXB_REQUIRE(is_float_type(dtype) && is_float_type(weights_dtype), "moe_unpermute_backward: rows and weights must be fp32, bf16 or fp16");
  FLUXB_REQUIRE(nexperts >= 1, "moe_unpermute_backward: nexperts=%d invalid", nexperts);
  int rc = check_sort("moe_unpermute_backward", ntokens, topk, hidden);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(dout != nullptr && splits != nullptr && scatter_index != nullptr && weights != nullptr && (drows != nullptr || dweights != nullptr),
                "moe_unpermute_backward: NULL argument");
  FLUXB_REQUIRE((rows != nullptr) == (dweights != nullptr), "moe_unpermute_backward: the weights' gradient needs the rows, and nothing else does");
  const int eb = dtype_bytes(dtype);
  const long long row_bytes = static_cast<long long>(hidden) * eb;
  const int vb = sort_vec_bytes(row_bytes, eb, {dout, rows, drows});
  const int row_vecs = static_cast<int>(row_bytes / vb);
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLUXB_CALL(T, VB) \
  launch_unpermute_backward<T, VB>(dout, rows, ntokens, topk, row_vecs, splits, nexperts, scatter_index, weights, weights_dtype, drows, dweights, s)
  FLUXB_SORT_TYPES(FLUXB_CALL);
#undef FLUXB_CALL
}

}  // extern "C"
