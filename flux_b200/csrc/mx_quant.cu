// Microscaled 4-bit floating point (the OCP MX format MXFP4): blocks of 32 values along K share one power of two.
//   s = floor(log2(max |x|)) - 2 (2: the exponent of e2m1's largest binade), at least -127, stored as s + 127;
//   q = x / 2^s rounded to the nearest of 0, 0.5, 1, 1.5, 2, 3, 4, 6 (ties to the even code), 6 at most.
// Dividing by the power of two is exact, so every q is the correctly rounded value. A block that holds an infinity or a
// NaN has the scale 255, which makes all of it NaN.
//
// Bound by memory, and by instructions next (75% of the issue slots with 8 values a thread and everything in fp32): two lanes
// share 32 values, 16 each, the largest is found in the input's own type, two values at a time, and bf16 is scaled so, too,
// which is exact. The four scales of a cell (mx_format.cuh) are one store. Two pieces of a thread are in flight together.
// 14336 x 12288 bf16 74 us, 6.0 TB/s (129 before); back to bf16 72 us, 6.2 TB/s (144 with codes taken apart by shifts).
#include "internal.h"
#include "mx_format.cuh"
#include "plain_gemm.cuh"

namespace fluxb {

constexpr int kQuantThreads = 256;
constexpr int kQuantUnroll = 2;
constexpr int kQuantUnit = 16;  // values of a thread at a time
constexpr int kQuantTailCtas = 148;  // at most: as many as a B200 has SMs
constexpr int kDequantUnroll = 4;

struct QuantParams {
  const void* x;
  long long ldx;       // elements between rows
  int rows, units;     // units in a row
  int groups;          // groups of 128 values in a row, started ones too: 8 units each
  FastDiv div;         // by 8 * groups
  FastDiv mat;         // by the rows of one matrix: every matrix starts a scale block
  int row0;            // first row of this launch
  uint8_t* data;
  uint8_t* scales;
  // quantised into the order of the experts: row t goes to the rows index[t, j]
  const int* index;
  const int* splits;
  int topk, nexperts, tail_ctas;  // (the first ones)
};

// row of the scale blocks that holds row r of the batch's matrices
__device__ __forceinline__ long long quant_scale_row(const FastDiv& mat, int r) {
  const int b = mat.quot(r);
  return b * ((static_cast<long long>(mat.d) + 127) & ~127ll) + (r - b * static_cast<int>(mat.d));
}

// 16 values of one of the input types, as words
template <class T>
struct QuantValues {
  static constexpr int W = 16 * sizeof(T) / 4;
  uint32_t w[W];
  __device__ __forceinline__ void load(const T* p, bool aligned) {
    if (aligned) {
#pragma unroll
      for (int i = 0; i < W / 4; ++i) {
        const uint4 v = __ldg(reinterpret_cast<const uint4*>(p) + i);
        w[4 * i] = v.x;
        w[4 * i + 1] = v.y;
        w[4 * i + 2] = v.z;
        w[4 * i + 3] = v.w;
      }
    } else if (sizeof(T) == 4) {
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = __float_as_uint(reinterpret_cast<const float*>(p)[i]);
    } else {
      const uint16_t* h = reinterpret_cast<const uint16_t*>(p);
#pragma unroll
      for (int i = 0; i < W; ++i) w[i] = h[2 * i] | (static_cast<uint32_t>(h[2 * i + 1]) << 16);
    }
  }
  __device__ __forceinline__ void clear() {
#pragma unroll
    for (int i = 0; i < W; ++i) w[i] = 0u;
  }
};
// Bits of the largest magnitude as a float's; magnitudes are compared as integers, where infinities and NaN come out on top.
__device__ __forceinline__ uint32_t quant_most16(const uint32_t (&w)[8]) {
  uint32_t m = w[0] & 0x7FFF7FFFu;
#pragma unroll
  for (int i = 1; i < 8; ++i) m = __vmaxu2(m, w[i] & 0x7FFF7FFFu);
  return max(m & 0xFFFFu, m >> 16);
}
__device__ __forceinline__ uint32_t quant_most(const QuantValues<float>& x) {
  uint32_t m = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) m = max(m, x.w[i] & 0x7FFFFFFFu);
  return m;
}
__device__ __forceinline__ uint32_t quant_most(const QuantValues<__nv_bfloat16>& x) { return quant_most16(x.w) << 16; }
__device__ __forceinline__ uint32_t quant_most(const QuantValues<__half>& x) {
  return __float_as_uint(__half2float(__ushort_as_half(static_cast<uint16_t>(quant_most16(x.w)))));
}
// The eight values from word 8 h (fp32) or 4 h on, times a power of two.
__device__ __forceinline__ void quant_scaled(const QuantValues<float>& x, int h, float inv, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 8; ++i) f[i] = __uint_as_float(x.w[8 * h + i]) * inv;
}
__device__ __forceinline__ void quant_scaled(const QuantValues<__nv_bfloat16>& x, int h, float inv, float (&f)[8]) {
  // exact: the products are at most 8, and those below bf16's normal numbers, which may be rounded, become zeros
  const __nv_bfloat162 s = __bfloat162bfloat162(__float2bfloat16_rn(inv));
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const __nv_bfloat162 v = __hmul2(*reinterpret_cast<const __nv_bfloat162*>(&x.w[4 * h + i]), s);
    const uint32_t b = *reinterpret_cast<const uint32_t*>(&v);
    f[2 * i] = __uint_as_float(b << 16);
    f[2 * i + 1] = __uint_as_float(b & 0xFFFF0000u);
  }
}
__device__ __forceinline__ void quant_scaled(const QuantValues<__half>& x, int h, float inv, float (&f)[8]) {
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 v = __half22float2(*reinterpret_cast<const __half2*>(&x.w[4 * h + i]));
    f[2 * i] = v.x * inv;
    f[2 * i + 1] = v.y * inv;
  }
}

// eight e2m1 codes, the first in the low bits
__device__ __forceinline__ uint32_t pack_e2m1(const float (&f)[8]) {
  uint32_t r;
  asm("{\n\t.reg .b8 a, b, c, d;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 a, %2, %1;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 b, %4, %3;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 c, %6, %5;\n\t"
      "cvt.rn.satfinite.e2m1x2.f32 d, %8, %7;\n\t"
      "mov.b32 %0, {a, b, c, d};\n\t}"
      : "=r"(r)
      : "f"(f[0]), "f"(f[1]), "f"(f[2]), "f"(f[3]), "f"(f[4]), "f"(f[5]), "f"(f[6]), "f"(f[7]));
  return r;
}

template <class T, bool SCATTER>
__global__ void __launch_bounds__(kQuantThreads)
mx_quantize_kernel(const __grid_constant__ QuantParams p, const int aligned) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (SCATTER && static_cast<int>(blockIdx.x) < p.tail_ctas) {
    // the rows that belong to no expert: zeros (8192 x 4096 top-2, a quarter dropped 21 us; by the last CTAs 26)
    __shared__ long long part[kQuantThreads / 32];
    long long s = 0;
    for (int e = threadIdx.x; e < p.nexperts; e += kQuantThreads) s += p.splits[e];
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) s += __shfl_xor_sync(0xffffffffu, s, off);
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = s;
    __syncthreads();
    s = 0;
#pragma unroll
    for (int w = 0; w < kQuantThreads / 32; ++w) s += part[w];
    if (s < 0) s = 0;
    const long long rows = static_cast<long long>(p.rows) * p.topk;
    for (long long r = s + blockIdx.x; r < rows; r += p.tail_ctas) {
      for (int u = threadIdx.x; u < p.units; u += kQuantThreads) reinterpret_cast<uint2*>(p.data)[r * p.units + u] = make_uint2(0u, 0u);
      for (int g = threadIdx.x; g < p.groups; g += kQuantThreads) *reinterpret_cast<uint32_t*>(p.scales + mx_sf_offset(r, g, p.groups)) = 0u;
    }
    return;
  }
  const int lane = threadIdx.x & 31;
  const int per_row = p.groups * 8;
  const int cta = static_cast<int>(blockIdx.x) - (SCATTER ? p.tail_ctas : 0);
  const long long u0 = static_cast<long long>(cta) * (kQuantThreads * kQuantUnroll) + threadIdx.x;
  QuantValues<T> in[kQuantUnroll];
  int row[kQuantUnroll], unit[kQuantUnroll];
#pragma unroll
  for (int i = 0; i < kQuantUnroll; ++i) {
    row[i] = p.div.quot(static_cast<int>(u0) + i * kQuantThreads);  // (past the last row: p.rows or more)
    unit[i] = static_cast<int>(u0) + i * kQuantThreads - row[i] * per_row;
    if (row[i] < p.rows && unit[i] < p.units) in[i].load(static_cast<const T*>(p.x) + row[i] * p.ldx + unit[i] * kQuantUnit, aligned != 0);
    else in[i].clear();
  }
#pragma unroll
  for (int i = 0; i < kQuantUnroll; ++i) {
    const bool valid = row[i] < p.rows && unit[i] < p.units;
    uint32_t most = quant_most(in[i]);
    most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
    const uint32_t field = most >> 23;
    uint2 code = make_uint2(0u, 0u);
    uint32_t scale = 255u;
    if (field != 255u) {
      scale = field < 2u ? 0u : field - 2u;
      const float inv = __uint_as_float((254u - scale) << 23);  // 2^(127 - scale), from 2^-125 to 2^127
      float f[8];
      quant_scaled(in[i], 0, inv, f);
      code.x = pack_e2m1(f);
      quant_scaled(in[i], 1, inv, f);
      code.y = pack_e2m1(f);
    }
    // the scales of 128 values (8 lanes, all of one row) as one word; those past the row's end are zero
    uint32_t cell = valid ? scale << (4 * (lane & 6)) : 0u;
    cell |= __shfl_xor_sync(0xffffffffu, cell, 2);
    cell |= __shfl_xor_sync(0xffffffffu, cell, 4);
    if (!valid) continue;
    const int kg = unit[i] >> 3;
    const bool writes_cell = (lane & 7) == 0;
    if (!SCATTER) {
      reinterpret_cast<uint2*>(p.data)[static_cast<long long>(p.row0 + row[i]) * p.units + unit[i]] = code;
      if (writes_cell) *reinterpret_cast<uint32_t*>(p.scales + mx_sf_offset(quant_scale_row(p.mat, p.row0 + row[i]), kg, p.groups)) = cell;
    } else {
      const int* idx = p.index + static_cast<long long>(row[i]) * p.topk;
      const long long rows = static_cast<long long>(p.rows) * p.topk;
      for (int j = 0; j < p.topk; ++j) {
        const long long r = __ldg(idx + j);
        if (r < 0 || r >= rows) continue;
        reinterpret_cast<uint2*>(p.data)[r * p.units + unit[i]] = code;
        if (writes_cell) *reinterpret_cast<uint32_t*>(p.scales + mx_sf_offset(r, kg, p.groups)) = cell;
      }
    }
  }
}

// Eight codes times their block's scale. Exact in fp32 (below 2^128), then one rounding to the output's type.
template <class T>
__device__ __forceinline__ T mx_out(float v);
template <>
__device__ __forceinline__ float mx_out(float v) { return v; }
template <>
__device__ __forceinline__ __nv_bfloat16 mx_out(float v) { return __float2bfloat16_rn(v); }
template <>
__device__ __forceinline__ __half mx_out(float v) { return __float2half_rn(v); }

template <class T>
__global__ void __launch_bounds__(kQuantThreads)
mx_dequantize_kernel(const uint32_t* __restrict__ data, const uint8_t* __restrict__ scales, int row0, int units, int groups, const FastDiv div,
                     const FastDiv mat, long long total, T* __restrict__ out) {
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  const long long u0 = static_cast<long long>(blockIdx.x) * (kQuantThreads * kDequantUnroll) + threadIdx.x;
  uint32_t code[kDequantUnroll], scale[kDequantUnroll];
#pragma unroll
  for (int i = 0; i < kDequantUnroll; ++i) {
    const long long u = u0 + i * kQuantThreads;
    if (u < total) {
      const int row = div.quot(static_cast<int>(u)), block = (static_cast<int>(u) - row * units) >> 2;
      code[i] = __ldg(data + u);
      scale[i] = __ldg(scales + mx_sf_offset(quant_scale_row(mat, row0 + row), block >> 2, groups) + (block & 3));
    }
  }
#pragma unroll
  for (int i = 0; i < kDequantUnroll; ++i) {
    const long long u = u0 + i * kQuantThreads;
    if (u >= total) break;
    const float s = scale[i] == 255u ? __uint_as_float(0x7FC00000u) : scale[i] == 0u ? __uint_as_float(0x00400000u) : __uint_as_float(scale[i] << 23);
    union {
      uint4 v[sizeof(T) / 2];
      T e[8];
    } o;
    uint32_t h[4];  // pairs of fp16, which holds every e2m1 value
    asm("{\n\t.reg .b8 a, b, c, d;\n\t"
        "mov.b32 {a, b, c, d}, %4;\n\t"
        "cvt.rn.f16x2.e2m1x2 %0, a;\n\t"
        "cvt.rn.f16x2.e2m1x2 %1, b;\n\t"
        "cvt.rn.f16x2.e2m1x2 %2, c;\n\t"
        "cvt.rn.f16x2.e2m1x2 %3, d;\n\t}"
        : "=r"(h[0]), "=r"(h[1]), "=r"(h[2]), "=r"(h[3])
        : "r"(code[i]));
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
      o.e[2 * j] = mx_out<T>(f.x * s);
      o.e[2 * j + 1] = mx_out<T>(f.y * s);
    }
#pragma unroll
    for (int j = 0; j < static_cast<int>(sizeof(T) / 2); ++j) reinterpret_cast<uint4*>(out + u * 8)[j] = o.v[j];
  }
}

static int mx_elt_bytes(int dt) { return dt == FLUXB_F32 ? 4 : dt == FLUXB_BF16 || dt == FLUXB_F16 ? 2 : 0; }

// Rows per launch: a unit's number is a 31-bit integer.
static int mx_rows_per_launch(int units) { return static_cast<int>(((1ll << 31) - kQuantThreads * kDequantUnroll - 1) / units); }

static int check_mx_matrices(const char* who, int batch, int rows, int k) {
  FLUXB_REQUIRE(batch >= 0 && rows >= 0 && k >= kMxBlock && k % kMxBlock == 0, "%s: batch=%d rows=%d k=%d invalid (k must be a multiple of %d)", who, batch,
                rows, k, kMxBlock);
  FLUXB_REQUIRE(static_cast<long long>(batch) * rows < (1ll << 31), "%s: %d x %d rows are too many", who, batch, rows);
  return FLUXB_OK;
}

}  // namespace fluxb

using namespace fluxb;

extern "C" {

int fluxb_mx_quantize(const void* x, int dtype, int batch, int rows, int k, long long ldx, void* data, void* scales, const int* splits_dev,
                      int nexperts, const int* scatter_index_dev, int topk, fluxb_stream_t stream) {
  const int eb = mx_elt_bytes(dtype);
  FLUXB_REQUIRE(eb != 0, "mx_quantize: the input must be fp32, bf16 or fp16");
  int rc = check_mx_matrices("mx_quantize", batch, rows, k);
  if (rc != FLUXB_OK) return rc;
  const bool scatter = scatter_index_dev != nullptr;
  FLUXB_REQUIRE(scatter == (splits_dev != nullptr), "mx_quantize: splits and scatter_index belong together");
  FLUXB_REQUIRE(!scatter || (batch == 1 && topk >= 1 && nexperts >= 1), "mx_quantize: batch=%d topk=%d nexperts=%d invalid", batch, topk, nexperts);
  FLUXB_REQUIRE(!scatter || static_cast<long long>(rows) * topk < (1ll << 30), "mx_quantize: too many routed rows");
  const int all = batch * rows;
  if (all == 0) return FLUXB_OK;
  FLUXB_REQUIRE(x != nullptr && data != nullptr && scales != nullptr, "mx_quantize: NULL argument");
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(x) & (eb - 1)) == 0 && (reinterpret_cast<uintptr_t>(data) & 7) == 0 && (reinterpret_cast<uintptr_t>(scales) & 3) == 0,
                "mx_quantize: the input must be aligned to its type, packed values to 8 bytes, scales to 4");
  FLUXB_REQUIRE(all_aligned(4, {splits_dev, scatter_index_dev}), "mx_quantize: splits and scatter_index must be aligned to their type");
  QuantParams p;
  memset(&p, 0, sizeof(p));
  p.ldx = ldx;
  p.units = k / kQuantUnit;
  p.groups = (k + kMxGroupK - 1) / kMxGroupK;
  p.div.set(static_cast<uint32_t>(p.groups) * 8u);
  p.mat.set(static_cast<uint32_t>(rows));
  p.data = static_cast<uint8_t*>(data);
  p.scales = static_cast<uint8_t*>(scales);
  p.index = scatter_index_dev;
  p.splits = splits_dev;
  p.topk = topk;
  p.nexperts = nexperts;
  const int most = mx_rows_per_launch(p.groups * 8);
  FLUXB_REQUIRE(!scatter || all <= most, "mx_quantize: too many values");
  const int aligned = ((reinterpret_cast<uintptr_t>(x) | static_cast<uintptr_t>(ldx * eb)) & 15) == 0 ? 1 : 0;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  for (long long r0 = 0; r0 < all; r0 += most) {
    p.row0 = static_cast<int>(r0);
    p.x = static_cast<const uint8_t*>(x) + r0 * ldx * eb;
    p.rows = all - r0 < most ? static_cast<int>(all - r0) : most;
    const long long total = static_cast<long long>(p.rows) * p.groups * 8;
    const long long out_rows = static_cast<long long>(rows) * topk;
    p.tail_ctas = !scatter ? 0 : out_rows < kQuantTailCtas ? static_cast<int>(out_rows) : kQuantTailCtas;
    const int grid = p.tail_ctas + static_cast<int>((total + kQuantThreads * kQuantUnroll - 1) / (kQuantThreads * kQuantUnroll));
#define FLUXB_QUANTIZE(T) \
  (scatter ? launch_pdl(mx_quantize_kernel<T, true>, grid, kQuantThreads, s, p, aligned) : launch_pdl(mx_quantize_kernel<T, false>, grid, kQuantThreads, s, p, aligned))
    rc = dtype == FLUXB_F32 ? FLUXB_QUANTIZE(float) : dtype == FLUXB_BF16 ? FLUXB_QUANTIZE(__nv_bfloat16) : FLUXB_QUANTIZE(__half);
#undef FLUXB_QUANTIZE
    if (rc != FLUXB_OK) return rc;
  }
  return FLUXB_OK;
}

int fluxb_mx_dequantize(const void* data, const void* scales, int batch, int rows, int k, int out_dtype, void* out, fluxb_stream_t stream) {
  const int eb = mx_elt_bytes(out_dtype);
  FLUXB_REQUIRE(eb != 0, "mx_dequantize: the output must be fp32, bf16 or fp16");
  int rc = check_mx_matrices("mx_dequantize", batch, rows, k);
  if (rc != FLUXB_OK) return rc;
  const int all = batch * rows;
  if (all == 0) return FLUXB_OK;
  FLUXB_REQUIRE(data != nullptr && scales != nullptr && out != nullptr, "mx_dequantize: NULL argument");
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(data) & 3) == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0,
                "mx_dequantize: the packed values must be 4-byte aligned, the output 16-byte");
  const int units = k / 8, groups = (k + kMxGroupK - 1) / kMxGroupK;
  const int most = mx_rows_per_launch(units);
  FastDiv div, mat;
  div.set(static_cast<uint32_t>(units));
  mat.set(static_cast<uint32_t>(rows));
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  const uint8_t* sc = static_cast<const uint8_t*>(scales);
  for (long long r0 = 0; r0 < all; r0 += most) {
    const long long total = (all - r0 < most ? all - r0 : most) * units;
    const uint32_t* d = static_cast<const uint32_t*>(data) + r0 * units;
    uint8_t* o = static_cast<uint8_t*>(out) + r0 * k * eb;
    const int grid = static_cast<int>((total + kQuantThreads * kDequantUnroll - 1) / (kQuantThreads * kDequantUnroll)), row0 = static_cast<int>(r0);
    rc = out_dtype == FLUXB_F32    ? launch_pdl(mx_dequantize_kernel<float>, grid, kQuantThreads, s, d, sc, row0, units, groups, div, mat, total, reinterpret_cast<float*>(o))
         : out_dtype == FLUXB_BF16 ? launch_pdl(mx_dequantize_kernel<__nv_bfloat16>, grid, kQuantThreads, s, d, sc, row0, units, groups, div, mat, total,
                                                reinterpret_cast<__nv_bfloat16*>(o))
                                   : launch_pdl(mx_dequantize_kernel<__half>, grid, kQuantThreads, s, d, sc, row0, units, groups, div, mat, total,
                                                reinterpret_cast<__half*>(o));
    if (rc != FLUXB_OK) return rc;
  }
  return FLUXB_OK;
}

}  // extern "C"
