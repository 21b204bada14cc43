// The token side of a MoE layer, each step with its gradient: the experts of every token and their weights (route), the
// tokens copied into the order of their experts (permute) and the weighted sum of a token's rows (unpermute). The last two
// are bound by memory; every sum is in fp32 and in a fixed order, so results do not change from run to run.
//
// `scatter_index` [ntokens, topk] holds the row of every (token, choice) pair, as fluxb_moe_scatter_index makes it: the
// valid entries are the rows 0 .. sum(splits) - 1, each once; an entry outside [0, ntokens * topk) is a pair without an
// expert and takes no part. The rows from sum(splits) on belong to nobody: what is written there is zero.
#include "internal.h"

namespace fluxb {

// ----------------------------------------------------------------------------------------------------------- route
// z: logits of a token. chosen = the topk largest (ties: the lower expert), w = softmax over the chosen ones:
//   w_j = exp(z_j - z_max) / sum_i exp(z_i - z_max),   dz_j = w_j (dw_j - sum_i w_i dw_i),   0 for the others.
// A group of G lanes per token, VPL logits a lane in registers as order-preserving integers. A choice is a maximum over the
// lanes, ties to the lower expert, and only the lane that held it looks for its next one. 16-bit logits leave room for the
// expert in the same word, so that one maximum finds both; for fp32 a vote finds the lowest lane (its experts are lower)
// that has the largest key. So that no lane idles a warp takes as many tokens as it can: 32768 x 8 bf16 top-2 2.8 us (a warp
// per token 9.0), 16384 x 64 bf16 top-6 4.4, 32768 x 128 fp32 top-8 17.7 (maxima over 64-bit pairs of key and expert 22.5).
// Bound by instructions where the tokens fill the GPU (32768 x 128: an instruction in 71% of the active cycles with 77% of the
// warps resident; they wait for their turn, 34%, and for a busy pipe, 27%, more than for shuffles, 8%), by the launch's start and end
// where its CTAs all fit at once (16384 x 64: a third of the warps, 32% of the SMs' throughput).
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
// The same for 16-bit logits, in the upper half of a word; in the lower half the expert, lower ones larger.
template <class T>
__device__ __forceinline__ uint32_t route_key16(T x, int expert) {
  const float v = to_f32(x);
  if (v == -INFINITY) return 0u;
  uint32_t u = *reinterpret_cast<const uint16_t*>(&x);
  if (v == 0.0f) u = 0u;
  u = (u & 0x8000u) ? ~u & 0xFFFFu : u | 0x8000u;
  if (v != v) u = 0xFFFFu;
  return (u << 16) | (0xFFFFu - static_cast<uint32_t>(expert));
}
template <class T>
__device__ __forceinline__ float route_value16(uint32_t key) {
  const uint32_t u = key >> 16;
  if (u == 0xFFFFu) return __uint_as_float(0x7FC00000u);
  const uint16_t bits = static_cast<uint16_t>((u & 0x8000u) ? u ^ 0x8000u : ~u);
  return to_f32(*reinterpret_cast<const T*>(&bits));
}

template <class T, int G, int VPL>
__global__ void __launch_bounds__(kRouteThreads)
moe_route_kernel(const T* __restrict__ logits, int ntokens, int nexperts, int topk, int vectors, int* __restrict__ chosen, float* __restrict__ weights) {
  constexpr bool PACKED = sizeof(T) == 2;
  const int lane = threadIdx.x & (G - 1);
  const int t = static_cast<int>((static_cast<long long>(blockIdx.x) * kRouteThreads + threadIdx.x) / G);
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const bool live = t < ntokens;  // (all lanes of a warp meet at the shuffles)
  const T* z = logits + static_cast<long long>(live ? t : 0) * nexperts;
  const int first = lane * VPL;  // this lane's experts
  uint32_t key[VPL];
  auto key_of = [&](T x, int e) -> uint32_t {
    if (e >= nexperts) return 0u;
    if constexpr (PACKED) return route_key16<T>(x, e);
    else return route_key(x);
  };
  constexpr int PER = 16 / static_cast<int>(sizeof(T));
  if (VPL % PER == 0 && vectors) {
#pragma unroll
    for (int i = 0; i < VPL / PER; ++i) {
      union {
        uint4 v;
        T e[PER];
      } x;
      x.v = first + i * PER < nexperts ? __ldg(reinterpret_cast<const uint4*>(z + first) + i) : make_uint4(0u, 0u, 0u, 0u);
#pragma unroll
      for (int j = 0; j < PER; ++j) key[i * PER + j] = key_of(x.e[j], first + i * PER + j);
    }
  } else {
#pragma unroll
    for (int i = 0; i < VPL; ++i) key[i] = key_of(first + i < nexperts ? z[first + i] : from_f32<T>(0.0f), first + i);
  }
  uint32_t best = 0;  // this lane's largest
  int at = 0;         // (fp32) where it is
  auto look = [&] {
    best = key[0];
    at = 0;
#pragma unroll
    for (int i = 1; i < VPL; ++i) {
      if constexpr (PACKED) {
        best = max(best, key[i]);
      } else if (key[i] > best) {
        best = key[i];
        at = i;
      }
    }
  };
  look();
  int mine = -1;  // lane j: choice j
  uint32_t mine_key = 0;
  for (int j = 0; j < topk; ++j) {
    uint32_t top = best;
#pragma unroll
    for (int off = G / 2; off > 0; off >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, off));
    int e;
    bool held;
    if constexpr (PACKED) {
      e = static_cast<int>(0xFFFFu - (top & 0xFFFFu));
      held = best == top && top != 0u;
    } else {
      const int group = static_cast<int>(threadIdx.x) & 31 & ~(G - 1);  // the group's first lane in its warp
      const unsigned has = __ballot_sync(0xffffffffu, best == top) >> group;
      const int from = group + __ffs(static_cast<int>(has)) - 1;
      e = __shfl_sync(0xffffffffu, first + at, from);
      held = (static_cast<int>(threadIdx.x) & 31) == from && top != 0u;
    }
    if (lane == j && top != 0u) {  // (0: nothing left that may be chosen)
      mine = e;
      mine_key = top;
    }
    if (held) {
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (first + i == e) key[i] = 0u;
      look();
    }
  }
  float v;
  if constexpr (PACKED) v = route_value16<T>(mine_key); else v = route_value(mine_key);
  const float top_v = __shfl_sync(0xffffffffu, v, 0, G);
  const float p = mine >= 0 ? expf(v - top_v) : 0.0f;
  float sum = p;
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, off);
  if (live && lane < topk) {
    const long long o = static_cast<long long>(t) * topk + lane;
    chosen[o] = mine;
    weights[o] = mine >= 0 ? p / sum : 0.0f;
  }
}

// The row is cleared, then lane j writes the gradient of choice j: ordered by the warp's barrier.
template <class T, int G>
__global__ void __launch_bounds__(kRouteThreads)
moe_route_backward_kernel(const float* __restrict__ dweights, const int* __restrict__ chosen, const float* __restrict__ weights,
                          int ntokens, int nexperts, int topk, int vectors, T* __restrict__ dlogits) {
  const int lane = threadIdx.x & (G - 1);
  const int t = static_cast<int>((static_cast<long long>(blockIdx.x) * kRouteThreads + threadIdx.x) / G);
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const bool live = t < ntokens;
  T* out = dlogits + static_cast<long long>(live ? t : 0) * nexperts;
  if (live) {
    if (vectors) {
      for (int i = lane; i < nexperts * static_cast<int>(sizeof(T)) / 16; i += G) reinterpret_cast<uint4*>(out)[i] = make_uint4(0u, 0u, 0u, 0u);
    } else {
      for (int e = lane; e < nexperts; e += G) out[e] = from_f32<T>(0.0f);
    }
  }
  int c = -1;
  float w = 0.0f, dw = 0.0f;
  if (live && lane < topk) {
    const long long o = static_cast<long long>(t) * topk + lane;
    c = chosen[o];
    if (c >= 0 && c < nexperts) {
      w = weights[o];
      dw = dweights[o];
    } else {
      c = -1;
    }
  }
  float s = w * dw;
#pragma unroll
  for (int off = G / 2; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
  __syncwarp();
  if (c >= 0) out[c] = from_f32<T>(w * (dw - s));
}

// ---------------------------------------------------------------------------------------------------- permute, unpermute
constexpr int kSortThreads = 256;
constexpr int kSortTailCtas = 148;  // the rows that belong to nobody are cleared by CTAs of their own, as many as a B200 has SMs at most

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

// A warp takes 32 * UN vectors of a token: each is read once and stored to the token's rows.
// 8192 x 4096 bf16 top-2 33 us, 6.1 TB/s; 512 x 7168 top-8 10.6 (with four vectors 12.3, with a power of two of threads a token
// 11.8); rows of odd length go two or one bytes at a time, four of them (4096 x 4097 bf16 top-2 24 us, 4.2 TB/s; two of them 39).
constexpr int permute_vectors(int vb) { return vb == 16 ? 2 : 4; }
template <int VB>
__global__ void __launch_bounds__(kSortThreads)
moe_permute_kernel(const typename RawVec<VB>::type* __restrict__ tokens, int ntokens, int topk, int row_vecs, int units, int tail_ctas,
                   const int* __restrict__ splits, int nexperts, const int* __restrict__ index,
                   typename RawVec<VB>::type* __restrict__ rows_out) {
  const long long rows = static_cast<long long>(ntokens) * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (static_cast<int>(blockIdx.x) < tail_ctas) {
    sort_clear_tail<VB>(rows_out, rows, row_vecs, splits, nexperts, static_cast<int>(blockIdx.x), tail_ctas);
    return;
  }
  constexpr int UN = permute_vectors(VB);
  const int unit = (static_cast<int>(blockIdx.x) - tail_ctas) * (kSortThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  const int t = unit / units;
  if (t >= ntokens) return;
  const int v0 = (unit - t * units) * (32 * UN) + (static_cast<int>(threadIdx.x) & 31);
  const auto* src = tokens + static_cast<long long>(t) * row_vecs;
  const int* idx = index + static_cast<long long>(t) * topk;
  typename RawVec<VB>::type x[UN];
#pragma unroll
  for (int u = 0; u < UN; ++u)
    if (v0 + u * 32 < row_vecs) x[u] = __ldg(src + v0 + u * 32);
  for (int j = 0; j < topk; ++j) {
    const int r = __ldg(idx + j);
    if (r < 0 || r >= rows) continue;
    auto* dst = rows_out + static_cast<long long>(r) * row_vecs;
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (v0 + u * 32 < row_vecs) dst[v0 + u * 32] = x[u];
  }
}

__device__ __forceinline__ float load_weight(const void* w, int dtype, long long i) {
  if (dtype == FLUXB_F32) return static_cast<const float*>(w)[i];
  if (dtype == FLUXB_BF16) return __bfloat162float(static_cast<const __nv_bfloat16*>(w)[i]);
  return __half2float(static_cast<const __half*>(w)[i]);
}

// What a thread gathers from several rows comes through shared memory, by asynchronous copies of its own that it waits for
// in order: no thread reads what another has copied, so there are no barriers, and what is on its way is bound by shared
// memory (about 190 KB an SM) instead of registers. An item is UN choices of VU vectors of one token; items follow each
// other, a ring of D items is in flight. Items of 128 bytes (one vector of two rows, 32 bytes, spent
// more on the way from item to item than on memory: 8192 x 4096 bf16 top-2 46 us).
constexpr int kGatherSmem = 96 * 1024;  // a CTA's share, two CTAs an SM
constexpr int gather_vectors(int vb, int un) { return (vb == 16 ? 8 : 16) / un; }
constexpr int gather_depth(int vb, int un) { return kGatherSmem / (kSortThreads * vb * un * gather_vectors(vb, un)); }
template <int VB>
__device__ __forceinline__ void copy_async(uint32_t dst, const void* src) {
  if constexpr (VB == 16)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
  else
    asm volatile("cp.async.ca.shared.global [%0], [%1], 8;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void copy_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void copy_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
template <int VB>
__device__ __forceinline__ typename RawVec<VB>::type read_shared(uint32_t addr) {
  typename RawVec<VB>::type v;
  if constexpr (VB == 16)
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(addr) : "memory");
  else
    asm volatile("ld.shared.v2.b32 {%0, %1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(addr) : "memory");
  return v;
}

// Where a thread is: token, first vector, first choice.
struct GatherAt {
  int t, v, j;
};
template <int UN>
__device__ __forceinline__ void gather_index(int (&r)[UN], const int* index, const GatherAt& at, int ntokens, int topk, int rows) {
#pragma unroll
  for (int u = 0; u < UN; ++u) {
    r[u] = at.t < ntokens && at.j + u < topk ? __ldg(index + static_cast<long long>(at.t) * topk + at.j + u) : -1;
    if (r[u] >= rows) r[u] = -1;
  }
}
template <int UN>
__device__ __forceinline__ void gather_weights(float (&w)[UN], const void* weights, int wdtype, const GatherAt& at, int ntokens, int topk) {
#pragma unroll
  for (int u = 0; u < UN; ++u)
    w[u] = weights != nullptr && at.t < ntokens && at.j + u < topk ? load_weight(weights, wdtype, static_cast<long long>(at.t) * topk + at.j + u) : 1.0f;
}

// out[t] = sum_j w[t, j] rows[index[t, j]], j ascending, rounded once; without weights the plain sum.
// 8192 x 4096 bf16 top-2 32 us, 6.3 TB/s (one vector of two rows a thread and a CTA for every token 60, eight vectors in
// registers and resident CTAs 38); 8192 x 2048 top-6 39 us, 6.0 TB/s (72, 65; eight choices an item 46). Rows are shared out by
// the warp's 32 * VU vectors: as many threads to a token as a power of two has left half of them without work where a row is a
// little longer (8192 x 4100 top-2 34 us against 44, 8192 x 2052 top-6 45 against 82, 2000 x 5120 fp16 top-4 18 against 20).
template <class T, int VB, int UN>
__global__ void __launch_bounds__(kSortThreads, 2)
moe_unpermute_kernel(const typename RawVec<VB>::type* __restrict__ rows_in, int ntokens, int topk, int row_vecs,
                     const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                     typename RawVec<VB>::type* __restrict__ out) {
  using V = SortVec<T, VB>;
  constexpr int VU = gather_vectors(VB, UN), D = gather_depth(VB, UN);
  extern __shared__ __align__(16) uint8_t gather_smem[];
  const uint32_t slots = smem_u32(gather_smem) + threadIdx.x * VB;  // [D][UN][VU][threads] vectors
  const int rows = ntokens * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  // a warp's units: 32 * VU vectors of a token, units of all tokens one after the other
  const int unit = 32 * VU, units = (row_vecs + unit - 1) / unit, all_vecs = units * unit;
  const int start = static_cast<int>(blockIdx.x) * (kSortThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  const int step = static_cast<int>(gridDim.x) * (kSortThreads / 32), step_t = step / units, step_v = (step - step_t * units) * unit;
  auto next = [&](GatherAt& at) {  // choices change fastest
    at.j += UN;
    if (at.j < topk) return;
    at.j = 0;
    at.t += step_t;
    at.v += step_v;
    if (at.v < all_vecs) return;
    at.v -= all_vecs;
    ++at.t;
  };
  GatherAt put{start / units, start % units * unit + (static_cast<int>(threadIdx.x) & 31), 0};
  GatherAt get = put, ahead = put;
  int row[UN];
  gather_index<UN>(row, index, put, ntokens, topk, rows);
  int stage_put = 0;
  auto issue = [&] {
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (row[u] >= 0) {
        const auto* src = rows_in + static_cast<long long>(row[u]) * row_vecs + put.v;
#pragma unroll
        for (int k = 0; k < VU; ++k)
          if (put.v + k * 32 < row_vecs) copy_async<VB>(slots + ((stage_put * UN + u) * VU + k) * (kSortThreads * VB), src + k * 32);
      }
    copy_commit();
    if (++stage_put == D) stage_put = 0;
    next(put);
    gather_index<UN>(row, index, put, ntokens, topk, rows);
  };
#pragma unroll 1
  for (int i = 0; i < D - 1; ++i) issue();
  int cur[UN], nxt[UN];
  float w[UN], nxt_w[UN];
  gather_index<UN>(nxt, index, ahead, ntokens, topk, rows);
  gather_weights<UN>(nxt_w, weights, wdtype, ahead, ntokens, topk);
  float acc[VU][V::N];
  int stage = 0;
  while (get.t < ntokens) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      cur[u] = nxt[u];
      w[u] = nxt_w[u];
    }
    next(ahead);
    gather_index<UN>(nxt, index, ahead, ntokens, topk, rows);
    gather_weights<UN>(nxt_w, weights, wdtype, ahead, ntokens, topk);
    issue();
    copy_wait<D - 1>();
    if (get.j == 0) {
#pragma unroll
      for (int k = 0; k < VU; ++k)
#pragma unroll
        for (int i = 0; i < V::N; ++i) acc[k][i] = 0.0f;
    }
#pragma unroll
    for (int u = 0; u < UN; ++u)
      if (cur[u] >= 0) {
#pragma unroll
        for (int k = 0; k < VU; ++k) {
          V x;  // (vectors past the row's end were not copied, and are not stored)
          x.raw = read_shared<VB>(slots + ((stage * UN + u) * VU + k) * (kSortThreads * VB));
#pragma unroll
          for (int i = 0; i < V::N; ++i) acc[k][i] = fmaf(w[u], to_f32(x.e[i]), acc[k][i]);
        }
      }
    if (get.j + UN >= topk) {
#pragma unroll
      for (int k = 0; k < VU; ++k)
        if (get.v + k * 32 < row_vecs) {
          V y;
#pragma unroll
          for (int i = 0; i < V::N; ++i) y.e[i] = from_f32<T>(acc[k][i]);
          out[static_cast<long long>(get.t) * row_vecs + get.v + k * 32] = y.raw;
        }
    }
    if (++stage == D) stage = 0;
    next(get);
  }
  copy_wait<0>();
}

// The same for vectors of 2 and 4 bytes (odd row lengths), with UN rows of VU vectors in registers: asynchronous copies do
// not know 2 bytes, and take an instruction for every 4. 16 vectors in flight (8 or 32 are slower): 4096 x 4097 bf16 top-2 25 us,
// 4.0 TB/s; 4096 x 2049 fp16 top-8 43 (a token at a time by a power of two of threads, 8 vectors 39 and 83).
template <class T, int VB, int UN, int VU>
__global__ void __launch_bounds__(kSortThreads)
moe_unpermute_narrow_kernel(const typename RawVec<VB>::type* __restrict__ rows_in, int ntokens, int topk, int row_vecs,
                            const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                            typename RawVec<VB>::type* __restrict__ out) {
  using V = SortVec<T, VB>;
  const int rows = ntokens * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const int unit = 32 * VU, units = (row_vecs + unit - 1) / unit, all_vecs = units * unit;
  const int start = static_cast<int>(blockIdx.x) * (kSortThreads / 32) + (static_cast<int>(threadIdx.x) >> 5);
  const int step = static_cast<int>(gridDim.x) * (kSortThreads / 32), step_t = step / units, step_v = (step - step_t * units) * unit;
  GatherAt at{start / units, start % units * unit + (static_cast<int>(threadIdx.x) & 31), 0};
  int row[UN], nxt[UN];
  float w[UN], nxt_w[UN];
  gather_index<UN>(nxt, index, at, ntokens, topk, rows);
  gather_weights<UN>(nxt_w, weights, wdtype, at, ntokens, topk);
  while (at.t < ntokens) {
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      row[u] = nxt[u];
      w[u] = nxt_w[u];
    }
    const int t = at.t, v0 = at.v;
    at.t += step_t;
    at.v += step_v;
    if (at.v >= all_vecs) {
      at.v -= all_vecs;
      ++at.t;
    }
    gather_index<UN>(nxt, index, at, ntokens, topk, rows);
    gather_weights<UN>(nxt_w, weights, wdtype, at, ntokens, topk);
    float acc[VU][V::N];
#pragma unroll
    for (int k = 0; k < VU; ++k)
#pragma unroll
      for (int i = 0; i < V::N; ++i) acc[k][i] = 0.0f;
    for (int j0 = 0; j0 < topk; j0 += UN) {
      if (topk > UN) {
        const GatherAt more{t, 0, j0};
        gather_index<UN>(row, index, more, ntokens, topk, rows);
        gather_weights<UN>(w, weights, wdtype, more, ntokens, topk);
      }
      V x[UN][VU];
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int k = 0; k < VU; ++k)
          if (row[u] >= 0 && v0 + k * 32 < row_vecs) x[u][k].raw = __ldg(rows_in + static_cast<long long>(row[u]) * row_vecs + v0 + k * 32);
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (row[u] >= 0) {
#pragma unroll
          for (int k = 0; k < VU; ++k)
#pragma unroll
            for (int i = 0; i < V::N; ++i) acc[k][i] = fmaf(w[u], to_f32(x[u][k].e[i]), acc[k][i]);
        }
    }
#pragma unroll
    for (int k = 0; k < VU; ++k)
      if (v0 + k * 32 < row_vecs) {
        V y;
#pragma unroll
        for (int i = 0; i < V::N; ++i) y.e[i] = from_f32<T>(acc[k][i]);
        out[static_cast<long long>(t) * row_vecs + v0 + k * 32] = y.raw;
      }
  }
}

// drows[index[t, j]] = w[t, j] dout[t] and dw[t, j] = <dout[t], rows[index[t, j]]>, KC choices at a time, whose rows and dout come
// through the ring: dout is read once for them, and the products stay in fp32 until the token's threads add them up.
// `rows_in` and `dweights` are null where only drows is wanted. An item is VU vectors; vectors change fastest, then choices.
// 8192 x 4096 bf16 top-2 56.5 us, 5.9 TB/s; 8192 x 2048 top-6 76 us, 5.7 TB/s (with the rows in registers 125).
constexpr int scatter_vectors(int kc) { return kc <= 4 ? 2 : 1; }
constexpr int scatter_depth(int vb, int kc) { return kGatherSmem / (kSortThreads * vb * (kc + 1) * scatter_vectors(kc)); }
template <class T, int VB, int KC>
__global__ void __launch_bounds__(kSortThreads, 2)
moe_unpermute_backward_kernel(const typename RawVec<VB>::type* __restrict__ dout, const typename RawVec<VB>::type* __restrict__ rows_in,
                              int ntokens, int topk, int row_vecs, int width, int main_ctas, const int* __restrict__ splits, int nexperts,
                              const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                              typename RawVec<VB>::type* __restrict__ drows, void* __restrict__ dweights) {
  using V = SortVec<T, VB>;
  constexpr int VU = scatter_vectors(KC), D = scatter_depth(VB, KC);
  __shared__ float part[2][kSortThreads / 32][KC];
  extern __shared__ __align__(16) uint8_t gather_smem[];
  const uint32_t slots = smem_u32(gather_smem) + threadIdx.x * VB;  // [D][KC + 1][VU][threads] vectors, dout first
  const int rows = ntokens * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (static_cast<int>(blockIdx.x) >= main_ctas) {
    if (drows != nullptr)
      sort_clear_tail<VB>(drows, rows, row_vecs, splits, nexperts, static_cast<int>(blockIdx.x) - main_ctas, static_cast<int>(gridDim.x) - main_ctas);
    return;
  }
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31, v_first = tid & (width - 1);
  const int per = kSortThreads / width, step = main_ctas * per;
  const int columns = (row_vecs + width * VU - 1) / (width * VU);  // items of a token and KC choices
  struct At {
    int t, j, c;
  };
  auto next = [&](At& at) {
    if (++at.c < columns) return;
    at.c = 0;
    at.j += KC;
    if (at.j < topk) return;
    at.j = 0;
    at.t += step;
  };
  auto choices = [&](int (&r)[KC], const At& at) { gather_index<KC>(r, index, GatherAt{at.t, 0, at.j}, ntokens, topk, rows); };
  At put{static_cast<int>(blockIdx.x) * per + tid / width, 0, 0}, get = put, ahead = put;
  int base = static_cast<int>(blockIdx.x) * per;  // the CTA's first token: all its threads meet at the sums
  int row[KC];
  choices(row, put);
  int stage_put = 0;
  auto issue = [&] {
    if (put.t < ntokens) {
#pragma unroll
      for (int k = 0; k < VU; ++k) {
        const int v = v_first + (put.c * VU + k) * width;
        if (v >= row_vecs) continue;
        const uint32_t dst = slots + (stage_put * (KC + 1) * VU + k) * (kSortThreads * VB);
        copy_async<VB>(dst, dout + static_cast<long long>(put.t) * row_vecs + v);
        if (rows_in != nullptr) {
#pragma unroll
          for (int u = 0; u < KC; ++u)
            if (row[u] >= 0) copy_async<VB>(dst + (u + 1) * VU * (kSortThreads * VB), rows_in + static_cast<long long>(row[u]) * row_vecs + v);
        }
      }
    }
    copy_commit();
    if (++stage_put == D) stage_put = 0;
    next(put);
    choices(row, put);
  };
#pragma unroll 1
  for (int i = 0; i < D - 1; ++i) issue();
  int cur[KC], nxt[KC];
  float w[KC], nxt_w[KC], dot[KC];
  choices(nxt, ahead);
  gather_weights<KC>(nxt_w, weights, wdtype, GatherAt{ahead.t, 0, ahead.j}, ntokens, topk);
  int stage = 0, turn = 0;
  while (base < ntokens) {
#pragma unroll
    for (int u = 0; u < KC; ++u) {
      cur[u] = nxt[u];
      w[u] = nxt_w[u];
      if (get.c == 0) dot[u] = 0.0f;
    }
    next(ahead);
    choices(nxt, ahead);
    gather_weights<KC>(nxt_w, weights, wdtype, GatherAt{ahead.t, 0, ahead.j}, ntokens, topk);
    issue();
    copy_wait<D - 1>();
#pragma unroll
    for (int k = 0; k < VU; ++k) {
      const int v = v_first + (get.c * VU + k) * width;
      if (v >= row_vecs) continue;
      const uint32_t src = slots + (stage * (KC + 1) * VU + k) * (kSortThreads * VB);
      V g;
      g.raw = read_shared<VB>(src);
#pragma unroll
      for (int u = 0; u < KC; ++u) {
        if (cur[u] < 0) continue;
        if (rows_in != nullptr) {
          V x;
          x.raw = read_shared<VB>(src + (u + 1) * VU * (kSortThreads * VB));
#pragma unroll
          for (int i = 0; i < V::N; ++i) dot[u] = fmaf(to_f32(g.e[i]), to_f32(x.e[i]), dot[u]);
        }
        if (drows != nullptr) {
          V d;
#pragma unroll
          for (int i = 0; i < V::N; ++i) d.e[i] = from_f32<T>(w[u] * to_f32(g.e[i]));
          drows[static_cast<long long>(cur[u]) * row_vecs + v] = d.raw;
        }
      }
    }
    if (++stage == D) stage = 0;
    if (get.c == columns - 1 && dweights != nullptr) {
#pragma unroll
      for (int u = 0; u < KC; ++u) {
#pragma unroll
        for (int off = 16; off > 0; off >>= 1) dot[u] += __shfl_xor_sync(0xffffffffu, dot[u], off);
        if (lane == 0) part[turn][warp][u] = dot[u];
      }
      __syncthreads();  // (one: the next sums go to the other half)
      if (get.t < ntokens && v_first < KC && get.j + v_first < topk) {
        float s = 0.0f;
        for (int k = 0; k < width / 32; ++k) s += part[turn][tid / width * (width / 32) + k][v_first];
        const long long o = static_cast<long long>(get.t) * topk + get.j + v_first;
        if (wdtype == FLUXB_F32) static_cast<float*>(dweights)[o] = s;
        else if (wdtype == FLUXB_BF16) static_cast<__nv_bfloat16*>(dweights)[o] = __float2bfloat16_rn(s);
        else static_cast<__half*>(dweights)[o] = __float2half_rn(s);
      }
      turn ^= 1;
    }
    const int t_before = get.t;
    next(get);
    base += get.t - t_before;
  }
  copy_wait<0>();
}

// The same for vectors below 16 bytes, KC choices of VU vectors in registers. Vectors of 8 bytes (widths that 8 does not divide) against
// the ring, which has to copy twice as often for the same bytes: 8192 x 4100 bf16 top-2 60 and 85 us, 8192 x 2052 top-6 91 and 133,
// 2000 x 5124 fp16 top-4 35 and 41. (The sum above reads only, and is faster from the ring: top-6 53 against 152.)
template <class T, int VB, int KC, int VU>
__global__ void __launch_bounds__(kSortThreads)
moe_unpermute_backward_narrow_kernel(const typename RawVec<VB>::type* __restrict__ dout, const typename RawVec<VB>::type* __restrict__ rows_in,
                                     int ntokens, int topk, int row_vecs, int width, int tail_ctas, const int* __restrict__ splits, int nexperts,
                                     const int* __restrict__ index, const void* __restrict__ weights, int wdtype,
                                     typename RawVec<VB>::type* __restrict__ drows, void* __restrict__ dweights) {
  using V = SortVec<T, VB>;
  __shared__ float part[kSortThreads / 32][KC];
  const long long rows = static_cast<long long>(ntokens) * topk;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (static_cast<int>(blockIdx.x) < tail_ctas) {
    sort_clear_tail<VB>(drows, rows, row_vecs, splits, nexperts, static_cast<int>(blockIdx.x), tail_ctas);
    return;
  }
  const int per = kSortThreads / width;
  const int tid = static_cast<int>(threadIdx.x), warp = tid >> 5, lane = tid & 31;
  const long long t = static_cast<long long>(static_cast<int>(blockIdx.x) - tail_ctas) * per + tid / width;
  const bool live = t < ntokens;  // (all threads of the CTA meet at the barriers)
  for (int j0 = 0; j0 < topk; j0 += KC) {
    int row[KC];
    float w[KC], dot[KC];
#pragma unroll
    for (int u = 0; u < KC; ++u) {
      int r = live && j0 + u < topk ? __ldg(index + t * topk + j0 + u) : -1;
      if (r >= rows) r = -1;
      row[u] = r;
      w[u] = r >= 0 ? load_weight(weights, wdtype, t * topk + j0 + u) : 0.0f;
      dot[u] = 0.0f;
    }
    if (live) {
      for (int v0 = tid & (width - 1); v0 < row_vecs; v0 += VU * width) {
        V g[VU], x[KC][VU];
#pragma unroll
        for (int k = 0; k < VU; ++k)
          if (v0 + k * width < row_vecs) g[k].raw = __ldg(dout + t * row_vecs + v0 + k * width);
        if (rows_in != nullptr) {
#pragma unroll
          for (int u = 0; u < KC; ++u)
#pragma unroll
            for (int k = 0; k < VU; ++k)
              if (row[u] >= 0 && v0 + k * width < row_vecs) x[u][k].raw = __ldg(rows_in + static_cast<long long>(row[u]) * row_vecs + v0 + k * width);
        }
#pragma unroll
        for (int u = 0; u < KC; ++u) {
          if (row[u] < 0) continue;
#pragma unroll
          for (int k = 0; k < VU; ++k) {
            if (v0 + k * width >= row_vecs) continue;
            if (rows_in != nullptr) {
#pragma unroll
              for (int i = 0; i < V::N; ++i) dot[u] = fmaf(to_f32(g[k].e[i]), to_f32(x[u][k].e[i]), dot[u]);
            }
            if (drows != nullptr) {
              V d;
#pragma unroll
              for (int i = 0; i < V::N; ++i) d.e[i] = from_f32<T>(w[u] * to_f32(g[k].e[i]));
              drows[static_cast<long long>(row[u]) * row_vecs + v0 + k * width] = d.raw;
            }
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
// Threads per token that take `each` vectors of a row at a time.
static int sort_width(long long row_vecs, int each) {
  int w = 32;
  while (w < kSortThreads && static_cast<long long>(w) * each < row_vecs) w *= 2;
  return w;
}
// The same, or fewer, 64 at least, where that leaves the `ctas` that run side by side with less to do one after the other: rows a
// little longer than a power of two fill half of their places. Backward of 8192 x 4100 bf16 top-2 60 us (69 without), 8192 x 2052
// top-6 90 (103), 4096 x 1028 top-3 16 (25), but 4096 x 4098 fp32 top-2 61.5 (59.4); down to 32 threads that takes 66.5.
static int sort_width_even(int ntokens, long long row_vecs, int each, int ctas) {
  int w = sort_width(row_vecs, each);
  auto turns = [&](int width) {
    const long long at_once = static_cast<long long>(ctas) * (kSortThreads / width);
    return (ntokens + at_once - 1) / at_once * ((row_vecs + width * each - 1) / (width * each));
  };
  for (int fewer = w / 2; fewer >= 64; fewer /= 2)
    if (turns(fewer) < turns(w)) w = fewer;
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
  const T* z = static_cast<const T*>(logits);
  const int vectors = ((reinterpret_cast<uintptr_t>(logits) | static_cast<uintptr_t>(nexperts) * sizeof(T)) & 15) == 0 ? 1 : 0;
#define FLUXB_ROUTE(G, V)                                                                                                                            \
  if (nexperts <= G * V && topk <= G)                                                                                                                \
  return launch_pdl(moe_route_kernel<T, G, V>, static_cast<int>((static_cast<long long>(ntokens) * G + kRouteThreads - 1) / kRouteThreads), kRouteThreads, \
                    stream, z, ntokens, nexperts, topk, vectors, chosen, weights)
  FLUXB_ROUTE(8, 1);
  FLUXB_ROUTE(8, 4);
  FLUXB_ROUTE(8, 8);
  FLUXB_ROUTE(16, 8);
  FLUXB_ROUTE(16, 16);
  FLUXB_ROUTE(32, 8);
  FLUXB_ROUTE(32, 32);
#undef FLUXB_ROUTE
  FLUXB_FAIL(FLUXB_ERR_INVALID, "moe_route: nexperts=%d topk=%d not supported", nexperts, topk);
}

template <class T>
static int launch_route_backward(const float* dweights, const int* chosen, const float* weights, int ntokens, int nexperts, int topk, void* dlogits,
                                 cudaStream_t stream) {
  const int vectors = ((reinterpret_cast<uintptr_t>(dlogits) | static_cast<uintptr_t>(nexperts) * sizeof(T)) & 15) == 0 ? 1 : 0;
  const int g = topk <= 8 && nexperts <= 64 ? 8 : topk <= 16 && nexperts <= 256 ? 16 : 32;
  const int grid = static_cast<int>((static_cast<long long>(ntokens) * g + kRouteThreads - 1) / kRouteThreads);
  auto kern = g == 8 ? moe_route_backward_kernel<T, 8> : g == 16 ? moe_route_backward_kernel<T, 16> : moe_route_backward_kernel<T, 32>;
  return launch_pdl(kern, grid, kRouteThreads, stream, dweights, chosen, weights, ntokens, nexperts, topk, vectors, static_cast<T*>(dlogits));
}

// CTAs of `kern` with `smem` bytes that the current device holds at a time; `known` is the kernel's own
template <class Kern>
static int sort_resident_ctas(Kern kern, int smem, int (&known)[64], int* ctas) {
  int dev = 0;
  FLUXB_CUDA(cudaGetDevice(&dev));
  FLUXB_REQUIRE(dev < 64, "device index %d not supported", dev);
  if (known[dev] == 0) {
    int per_sm = 0, sms = 0;
    FLUXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    FLUXB_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, kern, kSortThreads, smem));
    FLUXB_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev));
    known[dev] = (per_sm > 0 ? per_sm : 1) * sms;
  }
  *ctas = known[dev];
  return FLUXB_OK;
}

template <class T, int VB, int UN>
static int launch_unpermute_rows(const void* rows, int ntokens, int topk, int row_vecs, const int* index, const void* weights, int wdtype, void* out,
                                 cudaStream_t stream) {
  using R = typename RawVec<VB>::type;
  static int known[64] = {};
  int ctas = 0;
  if constexpr (VB < 8) {
    constexpr int VU = 16 / UN;
    auto kern = moe_unpermute_narrow_kernel<T, VB, UN, VU>;
    const int rc = sort_resident_ctas(kern, 0, known, &ctas);
    if (rc != FLUXB_OK) return rc;
    const long long warps = static_cast<long long>(ntokens) * ((row_vecs + 32 * VU - 1) / (32 * VU)), need = (warps + kSortThreads / 32 - 1) / (kSortThreads / 32);
    return launch_pdl(kern, need < ctas ? static_cast<int>(need) : ctas, kSortThreads, stream, static_cast<const R*>(rows), ntokens, topk, row_vecs, index, weights,
                      wdtype, static_cast<R*>(out));
  } else {
    constexpr int VU = gather_vectors(VB, UN), SMEM = gather_depth(VB, UN) * UN * VU * VB * kSortThreads;
    auto kern = moe_unpermute_kernel<T, VB, UN>;
    const int rc = sort_resident_ctas(kern, SMEM, known, &ctas);
    if (rc != FLUXB_OK) return rc;
    const long long warps = static_cast<long long>(ntokens) * ((row_vecs + 32 * VU - 1) / (32 * VU)), need = (warps + kSortThreads / 32 - 1) / (kSortThreads / 32);
    return launch_pdl_cluster(kern, need < ctas ? static_cast<int>(need) : ctas, kSortThreads, SMEM, 0, stream, static_cast<const R*>(rows), ntokens, topk,
                              row_vecs, index, weights, wdtype, static_cast<R*>(out));
  }
}
template <class T, int VB>
static int launch_unpermute(const void* rows, int ntokens, int topk, int row_vecs, const int* index, const void* weights, int wdtype, void* out,
                            cudaStream_t stream) {
  if (topk <= 2) return launch_unpermute_rows<T, VB, 2>(rows, ntokens, topk, row_vecs, index, weights, wdtype, out, stream);
  return launch_unpermute_rows<T, VB, 4>(rows, ntokens, topk, row_vecs, index, weights, wdtype, out, stream);
}

template <class T, int VB, int KC>
static int launch_unpermute_backward_rows(const void* dout, const void* rows, int ntokens, int topk, int row_vecs, const int* splits, int nexperts,
                                          const int* index, const void* weights, int wdtype, void* drows, void* dweights, cudaStream_t stream) {
  using R = typename RawVec<VB>::type;
  constexpr bool NARROW = VB < 16;
  constexpr int VU = NARROW ? 8 / KC : scatter_vectors(KC), SMEM = NARROW ? 0 : scatter_depth(VB, KC) * (KC + 1) * VU * VB * kSortThreads;
  auto kern = [] {
    if constexpr (NARROW) return moe_unpermute_backward_narrow_kernel<T, VB, KC, VU>;
    else return moe_unpermute_backward_kernel<T, VB, KC>;
  }();
  static int known[64] = {};
  int ctas = 0;
  const int rc = sort_resident_ctas(kern, SMEM, known, &ctas);
  if (rc != FLUXB_OK) return rc;
  const int width = NARROW ? sort_width_even(ntokens, row_vecs, VU, ctas) : sort_width(row_vecs, VU), per = kSortThreads / width;
  const long long total = static_cast<long long>(ntokens) * topk;
  const int need = (ntokens + per - 1) / per, main_ctas = NARROW || need < ctas ? need : ctas;
  const int tail = drows == nullptr ? 0 : total < kSortTailCtas ? static_cast<int>(total) : kSortTailCtas;
  return launch_pdl_cluster(kern, main_ctas + tail, kSortThreads, SMEM, 0, stream, static_cast<const R*>(dout), static_cast<const R*>(rows), ntokens, topk, row_vecs,
                            width, NARROW ? tail : main_ctas, splits, nexperts, index, weights, wdtype, static_cast<R*>(drows), dweights);
}
template <class T, int VB>
static int launch_unpermute_backward(const void* dout, const void* rows, int ntokens, int topk, int row_vecs, const int* splits, int nexperts,
                                     const int* index, const void* weights, int wdtype, void* drows, void* dweights, cudaStream_t stream) {
  if (topk <= 2) return launch_unpermute_backward_rows<T, VB, 2>(dout, rows, ntokens, topk, row_vecs, splits, nexperts, index, weights, wdtype, drows, dweights, stream);
  if (topk <= 4) return launch_unpermute_backward_rows<T, VB, 4>(dout, rows, ntokens, topk, row_vecs, splits, nexperts, index, weights, wdtype, drows, dweights, stream);
  return launch_unpermute_backward_rows<T, VB, 8>(dout, rows, ntokens, topk, row_vecs, splits, nexperts, index, weights, wdtype, drows, dweights, stream);
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
  FLUXB_REQUIRE(all_aligned(dtype_bytes(dtype), {logits}) && all_aligned(4, {chosen_out, weights_out}), "moe_route: arguments must be aligned to their types");
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
  FLUXB_REQUIRE(all_aligned(dtype_bytes(dtype), {dlogits}) && all_aligned(4, {dweights, chosen, weights}),
                "moe_route_backward: arguments must be aligned to their types");
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  if (dtype == FLUXB_F32) return launch_route_backward<float>(dweights, chosen, weights, ntokens, nexperts, topk, dlogits, s);
  if (dtype == FLUXB_BF16) return launch_route_backward<__nv_bfloat16>(dweights, chosen, weights, ntokens, nexperts, topk, dlogits, s);
  return launch_route_backward<__half>(dweights, chosen, weights, ntokens, nexperts, topk, dlogits, s);
}

int fluxb_moe_permute(const void* tokens, int ntokens, int topk, long long row_bytes, const int* splits, int nexperts, const int* scatter_index,
                      void* rows_out, fluxb_stream_t stream) {
  FLUXB_REQUIRE(row_bytes >= 1 && row_bytes < (1ll << 30), "moe_permute: row_bytes=%lld invalid", row_bytes);
  FLUXB_REQUIRE(nexperts >= 1, "moe_permute: nexperts=%d invalid", nexperts);
  int rc = check_sort("moe_permute", ntokens, topk, 1);
  if (rc != FLUXB_OK) return rc;
  if (ntokens == 0) return FLUXB_OK;
  FLUXB_REQUIRE(tokens != nullptr && splits != nullptr && scatter_index != nullptr && rows_out != nullptr, "moe_permute: NULL argument");
  FLUXB_REQUIRE(all_aligned(4, {splits, scatter_index}), "moe_permute: arguments must be aligned to their types");
  const int vb = sort_vec_bytes(row_bytes, 1, {tokens, rows_out});
  const long long row_vecs = row_bytes / vb;
  const long long units = (row_vecs + 32 * permute_vectors(vb) - 1) / (32 * permute_vectors(vb)), warps = units * ntokens;
  FLUXB_REQUIRE(warps < (1ll << 31) - 8, "moe_permute: %d rows of %lld bytes are too many", ntokens, row_bytes);
  const long long total = static_cast<long long>(ntokens) * topk;
  const int tail = total < kSortTailCtas ? static_cast<int>(total) : kSortTailCtas;  // (first: they work beside the others)
  const int grid = tail + static_cast<int>((warps + kSortThreads / 32 - 1) / (kSortThreads / 32));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
#define FLUXB_PERMUTE(VB)                                                                                                                       \
  return launch_pdl(moe_permute_kernel<VB>, grid, kSortThreads, s, static_cast<const RawVec<VB>::type*>(tokens), ntokens, topk,                  \
                    static_cast<int>(row_vecs), static_cast<int>(units), tail, splits, nexperts, scatter_index, static_cast<RawVec<VB>::type*>(rows_out))
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
  FLUXB_REQUIRE(all_aligned(eb, {rows, out}) && all_aligned(4, {scatter_index}) && (weights == nullptr || all_aligned(dtype_bytes(weights_dtype), {weights})),
                "moe_unpermute: arguments must be aligned to their types");
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
  FLUXB_REQUIRE(all_aligned(eb, {dout, rows, drows}) && all_aligned(4, {splits, scatter_index}) && all_aligned(dtype_bytes(weights_dtype), {weights, dweights}),
                "moe_unpermute_backward: arguments must be aligned to their types");
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
