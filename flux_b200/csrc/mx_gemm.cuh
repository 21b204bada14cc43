// GEMMs of microscaled 4-bit operands (e2m1 values, one power of two for every 32 along K):
//   D[m, n] = sum over k of x[m, k] w[n, k] = sum over blocks b of 2^(sx[m, b] + sw[n, b] - 254) * sum of the block's products
// The tensor cores apply the scales (kind::mxf4, scale vectors 2X: 32 values); products of e2m1 values are exact, sums are
// in fp32.
//
// Operands are swapped as in the few-row GEMM: the 128 (or, for a CTA pair, 256) rows of a UMMA are rows of the weight,
// its N dimension is the tokens, 16 to 256 of them: a tile is as narrow as there are tokens, the weights of an expert
// with few tokens are not multiplied with padding, and a ragged end costs columns instead of 128-row boxes.
//
// A stage holds 256 values of K of every row of the tile: 128 bytes (swizzled, TMA) and 8 scale bytes. The tensor cores
// want the scales in tensor memory, row r of a block of 128 in lane r % 32 of column r / 32, four scales a cell, in all four
// quadrants: what tcgen05.cp makes of 512 consecutive bytes. Scales are kept that way in memory, too (mx_format.cuh),
// so that a copy brings them and no thread touches them. That matters because shared memory is the bound of these
// kernels: a stage of a 256 x 256 pair tile is 512 clocks of tensor work, and 32 KB written by the copies and 32 KB read by
// the tensor cores take all of them at 128 bytes a clock; barriers and loads of other warps wait behind that. (With
// row-major scales that warps rearranged, through shared memory or by tcgen05.st, 8192 x 28672 x 8192 took 757 us at best,
// in tiles of 192.)
#pragma once
#include "gemm_kernel.cuh"
#include "mx_format.cuh"

namespace fluxb {

constexpr int kMxStageK = 256;  // values of K per stage: 128 bytes
constexpr int kMxMaxExperts = 1024;
constexpr int kMxEpiWarps = 8;

struct MxParams {
  CUtensorMap tmap_w;   // weights [rows_w, K / 2 bytes]: 128 rows x 128 bytes
  CUtensorMap tmap_x;   // tokens [rows_x, K / 2 bytes]: this CTA's share of a tile's tokens x 128 bytes
  CUtensorMap tmap_sw;  // scale blocks, a row for every 128 rows: 1 x 1024 bytes (two groups of K)
  CUtensorMap tmap_sx;  // ... for all blocks of a tile; grouped: every expert's rows start a block
  const uint8_t* sx;    // few-token kernel, grouped: the tokens' scale blocks in row order
  int rows_x;           // tokens
  int N, num_kb, groups;  // groups = ceil(K / 128)
  int n_tiles, m_tiles, band;
  int w_blocks;         // grouped: scale blocks of an expert's weights
  int nexperts;         // grouped: experts, else 0
  const int* splits;    // grouped: tokens per expert
  int out_type;
  void* out;
  long long ldo;
  const void* bias;     // [N] of the output's type, or null
  int out_blocks;       // 16-bit output, rows 16-byte aligned
  int split;            // few-token kernel: CTAs that share a tile's K
  unsigned long long timeout_ns;
  int* status;
};

// Instruction descriptor of kind::mxf4: e2m1 operands, e8m0 scales, K = 64. `sf` selects the pair of scales within the
// 32-bit cell that this instruction's 64 values of K use (0 or 2), for both operands.
__host__ __device__ constexpr uint32_t mx_idesc(uint32_t m, uint32_t n, uint32_t sf) {
  return (sf << 4) | (1u << 7) | (1u << 10) | ((n >> 3) << 17) | (1u << 23) | ((m >> 4) << 24) | (sf << 29);
}

// 512 bytes as 32 rows x 16 bytes without swizzle, groups of 8 rows 128 bytes apart
__device__ __forceinline__ uint64_t mx_sf_desc(uint32_t smem_addr) {
  return static_cast<uint64_t>((smem_addr & 0x3FFFFu) >> 4) | (static_cast<uint64_t>(1) << 16) | (static_cast<uint64_t>(128 >> 4) << 32) |
         (static_cast<uint64_t>(1) << 46);
}

template <bool CTA2>
__device__ __forceinline__ void mx_copy_sf(uint32_t taddr, uint64_t desc) {
  if (CTA2)
    asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
  else
    asm volatile("tcgen05.cp.cta_group::1.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

template <bool CTA2>
__device__ __forceinline__ void umma_mxf4(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t sfa, uint32_t sfb, uint32_t accumulate) {
  if (CTA2)
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::mxf4.block_scale.scale_vec::2X [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(accumulate), "r"(sfa), "r"(sfb)
        : "memory");
}

template <int BN, bool CTA2, bool GROUPED>
struct MxLayout {
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBRows = CTA2 ? BN / 2 : BN;
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kXBlocks = (BN + 127) / 128;  // scale blocks of the tokens: all of them, in both CTAs of a pair
  static constexpr int kSfOffset = kABytes + kBBytes;
  static constexpr int kStageBytes = kSfOffset + (1 + kXBlocks) * 2 * kMxSfBytes;
  static constexpr int kTableBytes = GROUPED ? (2 * kMxMaxExperts + 1) * 4 : 0;
  static constexpr int kEpiBytes = kMxEpiWarps * 1024;  // 16 tokens x 32 columns of 16 bits and their neighbours, per epilogue warp
  static constexpr int kStagesFit = (232448 - 2048 - kTableBytes - kEpiBytes) / kStageBytes;
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  // Tensor memory: two accumulators and the scales of kSlots stages (for each of a stage's two groups of K four columns of
  // the weights and four for every 128 tokens). 2 x 256 columns leave no room for scales: there the second accumulator
  // starts kOverlap columns early, on the last columns of the first, which the epilogue reads before all others.
  static constexpr int kSfCols = 2 * 4 * (1 + kXBlocks);
  static constexpr int kSlotsFit = BN == 256 ? 4 : (512 - 2 * BN) / kSfCols;
  static constexpr int kSlots = kSlotsFit > kStages ? kStages : kSlotsFit;
  static constexpr int kOverlap = BN == 256 ? kSlots * kSfCols : 0;
  static constexpr int kAcc1 = BN - kOverlap;            // first column of the second accumulator
  static constexpr int kSf = 2 * BN - kOverlap;          // ... of the scales
  static constexpr int kColsUsed = kSf + kSlots * kSfCols;
  static constexpr uint32_t kTmemCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static constexpr int kNumBars = 2 * kStages + 5;
  static constexpr int kEpiOffset = kStages * kStageBytes;
  static constexpr int kBarOffset = kEpiOffset + kEpiBytes;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kGroupOffset = kMiscOffset + 64;
  static constexpr int kTotal = kGroupOffset + kTableBytes + 1024;
  // Grouped tokens start anywhere in a scale block. Single CTAs have a warp that gathers their scales; for pairs, whose two
  // CTAs would have to hand them over, a launch before this one moves them (mx_regroup_kernel).
  static constexpr bool kGather = GROUPED && !CTA2;
  static constexpr int kThreads = 64 + 32 * kMxEpiWarps + (kGather ? 32 : 0);
  static_assert(kStageBytes % 1024 == 0 && kSlots >= 2 && kStages >= 3 && kColsUsed <= 512, "layout");
};

// One warp's walk over the experts, 32 at a time: first row and end of expert e0 + lane, its tiles of `bn` tokens, and the
// number of tiles up to its end. Splits that are negative or run past the rows that exist are cut, so that nothing outside
// is touched.
struct MxExperts {
  long long rows = 0;
  int tiles = 0;
  int first, end, tiles_end, tiles_mine;
  int ahead;  // the split of expert e0 + lane, loaded a step before it is used
  __device__ __forceinline__ MxExperts(const int* splits, int nexperts, int lane) { ahead = lane < nexperts ? splits[lane] : 0; }
  __device__ __forceinline__ void next(const int* splits, int nexperts, int rows_x, int bn, int e0, int lane) {
    long long m = ahead > 0 ? ahead : 0;
    ahead = e0 + 32 + lane < nexperts ? splits[e0 + 32 + lane] : 0;
    long long incl = m;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    const long long f = rows + incl - m, e = rows + incl;
    first = static_cast<int>(f < rows_x ? f : rows_x);
    end = static_cast<int>(e < rows_x ? e : rows_x);
    tiles_mine = (end - first + bn - 1) / bn;
    int ti = tiles_mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int t = __shfl_up_sync(0xffffffffu, ti, off);
      if (lane >= off) ti += t;
    }
    tiles_end = tiles + ti;
    rows += __shfl_sync(0xffffffffu, incl, 31);
    tiles += __shfl_sync(0xffffffffu, ti, 31);
  }
};

// One output tile: rows w_row ... of the weight matrix (column n0 of its expert), tokens [m0, m_end), and where their scale
// blocks are; x_col = columns (32 tokens each) of its first block that are before the tile.
struct MxTile {
  int n0, w_row, w_block, m0, m_end, x_block, x_col;
};
// A run of `m_tiles` token tiles x n_tiles weight tiles, in bands of `band` weight tiles whose tiles go along the tokens:
// the tiles in flight cover about as many rows of one operand as of the other.
__device__ __forceinline__ void mx_raster(int t, int n_tiles, int m_tiles, int band, int& n_idx, int& m_idx) {
  const int per = band * m_tiles;
  const int b = t / per, r = t - b * per;
  const int h = n_tiles - b * band < band ? n_tiles - b * band : band;
  m_idx = r / h;
  n_idx = b * band + r - m_idx * h;
}
struct MxGroups {  // of a grouped launch, in shared memory
  int *row_first, *tile_end;
};
template <int BN, bool GROUPED>
__device__ __forceinline__ bool mx_tile(const MxParams& p, int tile_rows, int t, const MxGroups& g, MxTile& out) {
  int n_idx, m_idx;
  if (!GROUPED) {
    if (t >= p.n_tiles * p.m_tiles) return false;
    mx_raster(t, p.n_tiles, p.m_tiles, p.band, n_idx, m_idx);
    out.n0 = out.w_row = n_idx * tile_rows;
    out.w_block = out.n0 >> 7;
    out.m0 = m_idx * BN;
    out.m_end = p.rows_x;
    out.x_block = out.m0 >> 7;
  } else {
    const int gt = t / p.n_tiles;
    int lo = 0, hi = p.nexperts;  // the expert whose token tiles hold this one
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (g.tile_end[mid] > gt) hi = mid; else lo = mid + 1;
    }
    if (lo == p.nexperts) return false;
    const int before = lo > 0 ? g.tile_end[lo - 1] : 0;
    mx_raster(t - before * p.n_tiles, p.n_tiles, g.tile_end[lo] - before, p.band, n_idx, m_idx);
    out.n0 = n_idx * tile_rows;
    out.w_row = lo * p.N + out.n0;
    out.w_block = lo * p.w_blocks + (out.n0 >> 7);
    out.m0 = g.row_first[lo] + m_idx * BN;
    out.m_end = g.row_first[lo + 1];
    out.x_block = before * ((BN + 127) / 128) + ((m_idx * BN) >> 7);  // (as mx_regroup_kernel lays them out)
  }
  out.x_col = ((m_idx * BN) & 127) >> 5;
  return true;
}

__device__ __forceinline__ float mx_bias(const MxParams& p, int n) {
  if (p.bias == nullptr || n >= p.N) return 0.0f;
  if (p.out_type == kOutF32) return static_cast<const float*>(p.bias)[n];
  const uint16_t b = static_cast<const uint16_t*>(p.bias)[n];
  return p.out_type == kOutBf16 ? __uint_as_float(static_cast<uint32_t>(b) << 16) : __half2float(__ushort_as_half(b));
}
__device__ __forceinline__ uint16_t mx_round16(float v, bool bf16) {
  return bf16 ? __bfloat16_as_ushort(__float2bfloat16_rn(v)) : __half_as_ushort(__float2half_rn(v));
}

// Column n of `cnt` tokens from m on: a warp's 32 lanes write 64 (or 128) contiguous bytes of one token at a time.
template <int CNT>
__device__ __forceinline__ void mx_store_column(const MxParams& p, const uint32_t (&r)[CNT], int m, int cnt, int n, float bias) {
  if (n >= p.N) return;
  if (p.out_type == kOutF32) {
    float* o = static_cast<float*>(p.out) + m * p.ldo + n;
#pragma unroll
    for (int j = 0; j < CNT; ++j)
      if (j < cnt) o[j * p.ldo] = __uint_as_float(r[j]) + bias;
  } else {
    const bool bf16 = p.out_type == kOutBf16;
    uint16_t* o = static_cast<uint16_t*>(p.out) + m * p.ldo + n;
#pragma unroll
    for (int j = 0; j < CNT; ++j)
      if (j < cnt) o[j * p.ldo] = mx_round16(__uint_as_float(r[j]) + bias, bf16);
  }
}

// The same for 16-bit outputs whose rows are 16-byte aligned. A lane has one column, and two bytes of a row are slow to store
// (8192 x 14336 x 2048 took 190 us, most of it waiting for stores): the warp exchanges 16 tokens x 32 columns through 1 KB of
// its own, two tokens' values in a word, so that a lane gets eight columns of two tokens. Pieces of 16 bytes are
// exchanged in every other row, which keeps the reads off each other's banks.
__device__ __forceinline__ void mx_store_block(const MxParams& p, const uint32_t (&r)[32], int m, int cnt, int n0, float bias, uint32_t buf, int lane) {
  const bool bf16 = p.out_type == kOutBf16;
  const int oct = lane & 3, pair = lane >> 2;
  const bool cols = n0 + oct * 8 < p.N;  // (a multiple of 8)
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h * 16 >= cnt) break;
    __syncwarp();
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const float a = __uint_as_float(r[h * 16 + 2 * j]) + bias, b = __uint_as_float(r[h * 16 + 2 * j + 1]) + bias;
      const uint32_t w = bf16 ? pack_bf16(a, b) : pack_f16(a, b);
      asm volatile("st.shared.b32 [%0], %1;" ::"r"(buf + j * 128 + ((((lane >> 2) ^ (j & 1)) << 4) | ((lane & 3) << 2))), "r"(w) : "memory");
    }
    __syncwarp();
    uint32_t w[8];
#pragma unroll
    for (int q = 0; q < 2; ++q)
      asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                   : "=r"(w[4 * q]), "=r"(w[4 * q + 1]), "=r"(w[4 * q + 2]), "=r"(w[4 * q + 3])
                   : "r"(buf + pair * 128 + (((2 * oct + q) ^ (pair & 1)) << 4))
                   : "memory");
    const int t = h * 16 + 2 * pair;
    uint16_t* o = static_cast<uint16_t*>(p.out) + (m + t) * p.ldo + n0 + oct * 8;
    if (cols && t < cnt)
      *reinterpret_cast<uint4*>(o) = make_uint4(__byte_perm(w[0], w[1], 0x5410), __byte_perm(w[2], w[3], 0x5410), __byte_perm(w[4], w[5], 0x5410),
                                                __byte_perm(w[6], w[7], 0x5410));
    if (cols && t + 1 < cnt)
      *reinterpret_cast<uint4*>(o + p.ldo) = make_uint4(__byte_perm(w[0], w[1], 0x7632), __byte_perm(w[2], w[3], 0x7632), __byte_perm(w[4], w[5], 0x7632),
                                                        __byte_perm(w[6], w[7], 0x7632));
  }
}

// The scales of a grouped tile's tokens for one stage: of rows lane, lane + 32, ... the cells of two groups of K, zero past
// the tile's tokens and past K; then as 16-byte pieces in the order of a scale block.
template <int BN>
__device__ __forceinline__ void mx_gather_scales(uint32_t (&w)[2][4], const MxParams& p, int m0, int m_end, int kb, int lane) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int kg = kb * 2 + g, r = m0 + q * 32 + lane;
      w[g][q] = q * 32 < BN && r < m_end && kg < p.groups ? __ldg(reinterpret_cast<const uint32_t*>(p.sx + mx_sf_offset(r, kg, p.groups))) : 0u;
    }
}
__device__ __forceinline__ void mx_put_scales(const uint32_t (&w)[2][4], uint32_t dst, int lane) {
#pragma unroll
  for (int g = 0; g < 2; ++g)
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + g * kMxSfBytes + lane * 16), "r"(w[g][0]), "r"(w[g][1]), "r"(w[g][2]), "r"(w[g][3])
                 : "memory");
}

// Persistent kernel. Warp 0: TMA; warp 1: tensor memory and UMMA; kMxEpiWarps epilogue warps, two per quadrant. Two
// accumulators: the epilogue of a tile overlaps the main loop of the next.
template <int BN, bool CTA2, bool GROUPED>
__global__ void __launch_bounds__(MxLayout<BN, CTA2, GROUPED>::kThreads, 1)
mx_gemm_kernel(const __grid_constant__ MxParams p) {
  using L = MxLayout<BN, CTA2, GROUPED>;
  constexpr int STAGES = L::kStages, SLOTS = L::kSlots;
  constexpr int TILE_N = CTA2 ? 2 * kBM : kBM;
  constexpr bool OVERLAP = L::kOverlap > 0;
  static_assert(L::kTotal <= 232448, "shared memory budget exceeded");

  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_base + L::kBarOffset;
  auto bar_full = [&](int s) { return bar_base + 8u * s; };
  auto bar_empty = [&](int s) { return bar_base + 8u * (STAGES + s); };
  auto bar_tfull = [&](int a) { return bar_base + 8u * (2 * STAGES + a); };
  auto bar_tempty = [&](int a) { return bar_base + 8u * (2 * STAGES + 2 + a); };
  const uint32_t bar_retired = bar_base + 8u * (2 * STAGES + 4);
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 8);
  MxGroups groups;
  groups.row_first = reinterpret_cast<int*>(smem + L::kGroupOffset);
  groups.tile_end = groups.row_first + kMxMaxExperts + 1;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int half = CTA2 ? static_cast<int>(cluster_ctarank()) : 0;
  const bool leader = half == 0;
  const int worker = CTA2 ? static_cast<int>(blockIdx.x) >> 1 : static_cast<int>(blockIdx.x);
  const int workers = CTA2 ? static_cast<int>(gridDim.x) >> 1 : static_cast<int>(gridDim.x);
  const AbortWord ab{s_abort, CTA2 ? mapa_u32(smem_u32(const_cast<int*>(s_abort)), static_cast<uint32_t>(half ^ 1)) : 0u};
  const uint64_t budget = p.timeout_ns;

  if (warp == 0 && elect_one()) {
    *s_abort = 0;
    for (int s = 0; s < STAGES; ++s) {
      mbar_init(bar_full(s), L::kGather ? 2 : 1);  // the copies, and the warp that gathers scales
      mbar_init(bar_empty(s), 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(bar_tfull(a), 1);
      mbar_init(bar_tempty(a), (CTA2 ? 2 : 1) * kMxEpiWarps);
    }
    mbar_init(bar_retired, 1);
    mbar_init_fence();
    tma_prefetch_desc(&p.tmap_w);
    tma_prefetch_desc(&p.tmap_x);
    tma_prefetch_desc(&p.tmap_sw);
    tma_prefetch_desc(&p.tmap_sx);
  }
  if (warp == 1) {
    if (CTA2) {
      tmem_alloc_2cta(smem_u32(tmem_holder), L::kTmemCols);
      tmem_relinquish_2cta();
    } else {
      tmem_alloc(smem_u32(tmem_holder), L::kTmemCols);
      tmem_relinquish();
    }
  }
  if (GROUPED && warp == 2) {
    pdl_wait();
    MxExperts x(p.splits, p.nexperts, lane);
    for (int e0 = 0; e0 < p.nexperts; e0 += 32) {
      x.next(p.splits, p.nexperts, p.rows_x, BN, e0, lane);
      if (e0 + lane < p.nexperts) {
        groups.row_first[e0 + lane] = x.first;
        groups.tile_end[e0 + lane] = x.tiles_end;
      }
    }
    if (lane == 0) groups.row_first[p.nexperts] = static_cast<int>(x.rows < p.rows_x ? x.rows : p.rows_x);
  }
  tc_fence_before();
  if (CTA2) cluster_sync_all(); else __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  pdl_wait();  // nothing before this line (but a grouped launch's table) reads global memory
  if (threadIdx.x == 0) pdl_trigger();

  if (warp == 0) {
    // ------------------------------------------------------------------ TMA
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      const uint32_t full0 = CTA2 ? mapa_u32(bar_full(0), 0) : bar_full(0);
      const bool arms = !CTA2 || leader;
      MxTile tl, next;
      int t = worker;
      bool more = mx_tile<BN, GROUPED>(p, TILE_N, t, groups, next);
      while (ok && more) {
        tl = next;
        const int wrow = tl.w_row + half * kBM, xrow = tl.m0 + half * L::kBRows;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (kb == p.num_kb - 1) more = mx_tile<BN, GROUPED>(p, TILE_N, t += workers, groups, next);  // (while a stage is awaited)
          if (!mbar_wait(bar_empty(stage), phase ^ 1u, ab, kStatusTimeoutSmemEmpty, budget)) {
            ok = false;
            break;
          }
          if (arms) mbar_arrive_expect_tx(bar_full(stage), (CTA2 ? 2 : 1) * (L::kStageBytes - (L::kGather ? 2 * L::kXBlocks * kMxSfBytes : 0)));
          const uint32_t fb = full0 + 8u * stage;
          const uint32_t sa = smem_base + stage * L::kStageBytes;
          auto load = [&](uint32_t dst, const void* map, int x, int y) {
            if (CTA2) tma_load_2d_2cta(dst, map, fb, x, y); else tma_load_2d(dst, map, fb, x, y);
          };
          load(sa, &p.tmap_w, kb * kRowBytes, wrow);
          load(sa + L::kABytes, &p.tmap_x, kb * kRowBytes, xrow);
          load(sa + L::kSfOffset, &p.tmap_sw, kb * 256, tl.w_block + half);
          if (!L::kGather) load(sa + L::kSfOffset + 2 * kMxSfBytes, &p.tmap_sx, kb * 256, tl.x_block);
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
      if (*s_abort != 0 && leader) {
        // every armed stage still has copies in flight or has been filled: wait (1 ms each at most)
        const AbortWord none{nullptr, 0u};
        for (int s2 = 0; s2 < STAGES; ++s2) mbar_wait(bar_full(s2), s2 < stage ? phase : (phase ^ 1u), none, 0, 1000000ull);
      }
    }
  } else if (warp == 1) {
    // ----------------------------------------------------------------- UMMA
    if (leader && elect_one()) {
      const uint64_t a_desc0 = make_kmajor_sw128_desc(smem_base), b_desc0 = make_kmajor_sw128_desc(smem_base + L::kABytes);
      const uint64_t sf_desc0 = mx_sf_desc(smem_base + L::kSfOffset);
      constexpr uint32_t UM = CTA2 ? 256 : 128;
      int stage = 0, slot = 0, it = 0, issued = 0;
      uint32_t phase = 0;
      int old_stage = 0;  // the stage that used this slot of scales last, and its phase
      uint32_t old_phase = 0;
      bool ok = true;
      MxTile tl;
      for (int t = worker; ok && mx_tile<BN, GROUPED>(p, TILE_N, t, groups, tl); t += workers, ++it) {
        const int acc = it & 1;
        // its accumulator has been read
        if (!OVERLAP && !mbar_wait<CTA2>(bar_tempty(acc), ((it >> 1) & 1) ^ 1u, ab, kStatusTimeoutTmemEmpty, budget)) break;
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * L::kAcc1);
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait(bar_full(stage), phase, ab, kStatusTimeoutSmemFull, budget)) {
            ok = false;
            break;
          }
          // the scales' columns are used again once the UMMAs that read them have retired
          if (SLOTS < STAGES) {
            if (issued == SLOTS) {
              if (!mbar_wait(bar_empty(old_stage), old_phase, ab, kStatusTimeoutSmemEmpty, budget)) {
                ok = false;
                break;
              }
              if (++old_stage == STAGES) {
                old_stage = 0;
                old_phase ^= 1u;
              }
            } else {
              ++issued;
            }
          }
          tc_fence_after();
          const uint32_t off = static_cast<uint32_t>(stage) * (L::kStageBytes >> 4);
          const uint32_t sf = tmem_base + static_cast<uint32_t>(L::kSf + slot * L::kSfCols);
          constexpr int GC = 4 * (1 + L::kXBlocks);  // columns per group of K
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int b = 0; b < 1 + L::kXBlocks; ++b)
              mx_copy_sf<CTA2>(sf + g * GC + b * 4, sf_desc0 + off + static_cast<uint32_t>((b * 2 + g) * (kMxSfBytes >> 4)));
          if (OVERLAP && kb == 0 && it > 0) {
            // the columns that the tile before shares with this one have been read (and with them everything of the tile before
            // that); the first stage's scales are on their way by then
            if (!mbar_wait<CTA2>(bar_tempty(0), (it - 1) & 1, ab, kStatusTimeoutTmemEmpty, budget)) {
              ok = false;
              break;
            }
            tc_fence_after();
          }
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t sfa = sf + (k >> 1) * GC;
            umma_mxf4<CTA2>(d, a_desc0 + off + 2u * k, b_desc0 + off + 2u * k, mx_idesc(UM, BN, (k & 1) * 2), sfa,
                            sfa + 4 + (BN % 128 == 0 || L::kGather ? 0 : tl.x_col), (kb > 0 || k > 0) ? 1u : 0u);
          }
          if (CTA2) umma_commit_2cta(bar_empty(stage), 3); else umma_commit(bar_empty(stage));
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
          if (++slot == SLOTS) slot = 0;
        }
        if (ok) {
          if (CTA2) umma_commit_2cta(bar_tfull(acc), 3); else umma_commit(bar_tfull(acc));
        }
      }
      if (*s_abort != 0) {  // UMMAs in flight still read shared memory and write tensor memory
        if (CTA2) umma_commit_2cta(bar_retired, 1); else umma_commit(bar_retired);
        mbar_wait(bar_retired, 0, AbortWord{nullptr, 0u}, 0, 2000000ull);
      }
    }
  } else if (warp < 2 + kMxEpiWarps) {
    // ------------------------------------------------------------- epilogue
    const int quad = warp & 3, first = (warp - 2) >> 2;
    const uint32_t tmem_quad = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
    const uint32_t tempty0 = CTA2 ? mapa_u32(bar_tempty(0), 0) : bar_tempty(0);
    const uint32_t epi_buf = smem_base + L::kEpiOffset + (warp - 2) * 1024;
    const bool blocks = p.out_blocks != 0;
    constexpr int CHUNKS = BN / 32, SHARED = L::kOverlap / 32;
    static_assert(BN % 32 == 0 && L::kOverlap % 32 == 0, "chunks");
    int it = 0;
    MxTile tl;
    for (int t = worker; mx_tile<BN, GROUPED>(p, TILE_N, t, groups, tl); t += workers, ++it) {
      const int acc = it & 1;
      const int n = tl.n0 + half * kBM + quad * 32 + lane;
      const float bias = mx_bias(p, n);
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull(acc), (it >> 1) & 1, ab, kStatusTimeoutTmemFull, budget, 100))) break;
      tc_fence_after();
      const uint32_t tacc = tmem_quad + static_cast<uint32_t>(acc * L::kAcc1);
      auto give_back = [&] {
        tc_fence_before();
        __syncwarp();
        if (lane == 0) {
          const uint32_t bar = tempty0 + (OVERLAP ? 0u : 8u * acc);
          if (CTA2) mbar_arrive_cluster(bar); else mbar_arrive(bar);
        }
      };
      auto store = [&](const uint32_t (&r)[32], int c) {
        if (blocks) mx_store_block(p, r, tl.m0 + c, tl.m_end - tl.m0 - c, n - lane, bias, epi_buf, lane);
        else mx_store_column<32>(p, r, tl.m0 + c, tl.m_end - tl.m0 - c, n, bias);
      };
      int i = first;
      if constexpr (OVERLAP) {
        // the columns that the next tile's accumulator shares, the last ones of the first and the first of the second, leave
        // tensor memory before anything is stored: the UMMAs of that tile wait for them
        static_assert(SHARED <= 4, "at most two chunks a warp");
        uint32_t r0[32], r1[32];
        const int c0 = (acc == 0 ? CHUNKS - 1 - first : first) * 32, c1 = (acc == 0 ? CHUNKS - 3 - first : first + 2) * 32;
        const bool two = first + 2 < SHARED;
        tmem_ld_32x32(tacc + c0, r0);
        if (two) tmem_ld_32x32(tacc + c1, r1);
        tmem_ld_wait();
        give_back();
        if (tl.m0 + c0 < tl.m_end) store(r0, c0);
        if (two && tl.m0 + c1 < tl.m_end) store(r1, c1);
        i += two ? 4 : 2;
      }
#pragma unroll 1
      for (; i < CHUNKS; i += 2) {
        const int c = (OVERLAP && acc == 0 ? CHUNKS - 1 - i : i) * 32;
        if (tl.m0 + c >= tl.m_end) continue;
        uint32_t r[32];
        tmem_ld_32x32(tacc + c, r);
        tmem_ld_wait();
        store(r, c);
      }
      if (!OVERLAP) give_back();
    }
  } else if constexpr (L::kGather) {
    // ------------------------------------------------ scales of grouped tokens
    // four stages at a time, the next four's words already on their way: a pair at a time, the warp's loads took as long as the
    // stages' copies (64 experts of 6 tokens x 2048 x 2048 33.3 us)
    static_assert(L::kXBlocks == 1, "one block of rows");
    constexpr int UN = 4;
    auto fetch = [&](uint32_t (&w)[UN][2][4], const MxTile& x, int kb) {
#pragma unroll
      for (int u = 0; u < UN; ++u) mx_gather_scales<BN>(w[u], p, x.m0, x.m_end, kb + u, lane);
    };
    int stage = 0, t = worker, kb = 0;
    uint32_t phase = 1;
    MxTile tl;
    uint32_t cur[UN][2][4], nxt[UN][2][4];
    bool more = mx_tile<BN, GROUPED>(p, TILE_N, t, groups, tl);
    if (more) fetch(cur, tl, 0);
    bool ok = true;
    while (more && ok) {
      const int n = p.num_kb - kb < UN ? p.num_kb - kb : UN;
      kb += UN;
      if (kb >= p.num_kb) {
        kb = 0;
        t += workers;
        more = mx_tile<BN, GROUPED>(p, TILE_N, t, groups, tl);
      }
      if (more) fetch(nxt, tl, kb);
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (u >= n || !ok) break;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_empty(stage), phase, ab, kStatusTimeoutSmemEmpty, budget))) {
          ok = false;
          break;
        }
        mx_put_scales(cur[u], smem_base + stage * L::kStageBytes + L::kSfOffset + 2 * kMxSfBytes, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_full(stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
#pragma unroll
      for (int u = 0; u < UN; ++u)
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int q = 0; q < 4; ++q) cur[u][g][q] = nxt[u][g][q];
    }
  }

  // ------------------------------------------------------------------ teardown
  if (CTA2) cluster_sync_all(); else __syncthreads();
  if (*s_abort != 0 && threadIdx.x == 0) {
    *reinterpret_cast<volatile int*>(p.status) = *s_abort;
    __threadfence_system();
  }
  if (warp == 1) {
    __syncwarp();
    tc_fence_after();
    if (CTA2) tmem_dealloc_2cta(tmem_base, L::kTmemCols); else tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

// The tokens' scale blocks of a grouped launch with tiles of `bn` tokens: every expert's rows from a block's start on, the
// expert's blocks where its tiles, each of as many blocks as it has starts of 128 rows, begin. A CTA per block, as many as
// the experts could need, and 8 groups of K; 16 bytes (four rows 32 apart) per thread.
constexpr int kMxRegroupThreads = 256, kMxRegroupGroups = kMxRegroupThreads / 32;
static __global__ void __launch_bounds__(kMxRegroupThreads)
mx_regroup_kernel(const uint8_t* __restrict__ src, int rows, int groups, int parts, int bn, const int* __restrict__ splits, int nexperts,
                  uint4* __restrict__ dst) {
  __shared__ int s_first, s_end;
  const int lane = threadIdx.x & 31;
  const int block = static_cast<int>(blockIdx.x) / parts, part = static_cast<int>(blockIdx.x) - block * parts;
  pdl_wait();
  if (threadIdx.x == 0) pdl_trigger();
  if (threadIdx.x < 32) {
    const int per = (bn + 127) / 128, tile = block / per;
    MxExperts x(splits, nexperts, lane);
    int first = 0, end = 0;
    for (int e0 = 0; e0 < nexperts; e0 += 32) {
      x.next(splits, nexperts, rows, bn, e0, lane);
      const unsigned has = __ballot_sync(0xffffffffu, x.tiles_end > tile);
      if (has == 0) continue;
      const int from = __ffs(has) - 1;
      const int before = __shfl_sync(0xffffffffu, x.tiles_end - x.tiles_mine, from);
      first = __shfl_sync(0xffffffffu, x.first, from) + (block - before * per) * 128;
      end = __shfl_sync(0xffffffffu, x.end, from);
      break;
    }
    if (lane == 0) {
      s_first = first;
      s_end = end;
    }
  }
  __syncthreads();
  const int first = s_first, end = s_end;
  if (first >= end) return;
  const int kg = part * kMxRegroupGroups + static_cast<int>(threadIdx.x >> 5);
  if (kg >= groups) return;
  uint32_t w[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = first + q * 32 + lane;
    w[q] = r < end ? __ldg(reinterpret_cast<const uint32_t*>(src + mx_sf_offset(r, kg, groups))) : 0u;
  }
  dst[(static_cast<long long>(block) * groups + kg) * 32 + lane] = make_uint4(w[0], w[1], w[2], w[3]);
}

// ------------------------------------------------------------------------------------------------------- few tokens
// Few tokens (up to 64, or a few per expert), where the time is that of reading the weights once and of getting started:
// one output tile per cluster of `split` CTAs, which cut K. Each CTA leaves its accumulator in its own shared memory; after
// a cluster barrier CTA r sums the tokens r * per ... of all parts, in rank order, through distributed shared memory: no
// scratch, no counters, any number of launches side by side. A grouped launch has a cluster for every tile that the
// experts could need (the counts are on the device); those that no expert needs leave at once. There a warp gathers the
// tokens' scales, whose rows start anywhere in a block.
constexpr int kMxFewThreads = 224;  // warp 0 TMA, warp 1 UMMA + tensor memory, warps 2-5 read-out and output, 6 scales of grouped tokens
constexpr int kMxFewMaxSplit = 8;
constexpr int kMxFewAhead = 3;  // K blocks of a CTA's weights that are fetched into the L2 ahead

template <int BN>
struct MxFewLayout {
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = BN * kRowBytes;
  static constexpr int kSfOffset = kABytes + kBBytes;
  static constexpr int kStageBytes = kSfOffset + 4 * kMxSfBytes;
  // a CTA takes half of an SM's shared memory, so that one CTA's prologue and reduction overlap another's loads
  static constexpr int kStages = BN == 16 ? 5 : 4;
  static_assert(BN <= 64 && kStages * kStageBytes >= BN * kBM * 4, "the read-out must fit into the stages");
  static constexpr int kSfCols = 16;
  static constexpr int kColsUsed = BN + kStages * kSfCols;
  static constexpr uint32_t kTmemCols = 128;
  static_assert(kColsUsed <= 128, "two CTAs' tensor memory");
  static constexpr int kNumBars = 2 * kStages + 2;  // full / empty per stage, accumulator complete, "UMMAs retired" (abort path)
  static constexpr int kBarOffset = kStages * kStageBytes;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 64 + 1024;  // + slack for 1024-byte alignment
};

// The tile of cluster `t` of a grouped launch, by one warp: the expert whose token tiles hold it. False: no expert has it.
template <int BN>
__device__ __forceinline__ bool mx_few_tile(const MxParams& p, int t, int lane, MxTile& out) {
  const int g = t / p.n_tiles;
  MxExperts x(p.splits, p.nexperts, lane);
  for (int e0 = 0; e0 < p.nexperts; e0 += 32) {
    x.next(p.splits, p.nexperts, p.rows_x, BN, e0, lane);
    const unsigned has = __ballot_sync(0xffffffffu, x.tiles_end > g);
    if (has == 0) continue;
    const int from = __ffs(has) - 1;
    const int before = __shfl_sync(0xffffffffu, x.tiles_end - x.tiles_mine, from);
    out.n0 = (t - g * p.n_tiles) * kBM;
    out.w_row = (e0 + from) * p.N + out.n0;
    out.w_block = (e0 + from) * p.w_blocks + (out.n0 >> 7);
    out.m0 = __shfl_sync(0xffffffffu, x.first, from) + (g - before) * BN;
    out.m_end = __shfl_sync(0xffffffffu, x.end, from);
    out.x_block = out.x_col = 0;
    return true;
  }
  return false;
}

// Output columns n, n + 1 of every second token of this CTA's share: the sum of the SPLIT parts in rank order, the bias,
// one rounding. UN tokens' loads are in flight together. A part that gave up leaves garbage here; its status word says so.
template <int SPLIT, int UN>
__device__ __forceinline__ void mx_few_reduce(const MxParams& p, uint32_t smem_base, const MxTile& tl, int cnt, int part, int t) {
  const int n = tl.n0 + (t & 63) * 2;
  if (n >= p.N) return;
  const int per = (cnt + SPLIT - 1) / SPLIT;
  const int m_end = imin(cnt, (part + 1) * per);
  uint32_t peer[SPLIT];
#pragma unroll
  for (int s = 0; s < SPLIT; ++s) peer[s] = mapa_u32(smem_base + (t & 63) * 8, s);
  const float b0 = mx_bias(p, n), b1 = mx_bias(p, n + 1);
  const bool both = n + 1 < p.N, paired = both && (p.ldo & 1) == 0 && (reinterpret_cast<uintptr_t>(p.out) & 3) == 0;
#pragma unroll 1
  for (int m0 = part * per + (t >> 6); m0 < m_end; m0 += 2 * UN) {
    uint2 v[UN][SPLIT];
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int m = m0 + 2 * u < m_end ? m0 + 2 * u : m0;
#pragma unroll
      for (int s = 0; s < SPLIT; ++s) v[u][s] = ld_shared_cluster_v2(peer[s] + static_cast<uint32_t>(m) * (kBM * 4));
    }
#pragma unroll
    for (int u = 0; u < UN; ++u) {
      const int m = m0 + 2 * u;
      if (m >= m_end) break;
      float x0 = __uint_as_float(v[u][0].x), x1 = __uint_as_float(v[u][0].y);
#pragma unroll
      for (int s = 1; s < SPLIT; ++s) {
        x0 += __uint_as_float(v[u][s].x);
        x1 += __uint_as_float(v[u][s].y);
      }
      x0 += b0;
      x1 += b1;
      const long long o = (tl.m0 + m) * p.ldo + n;
      if (p.out_type == kOutF32) {
        float* out = static_cast<float*>(p.out) + o;
        out[0] = x0;
        if (both) out[1] = x1;
      } else {
        const bool bf16 = p.out_type == kOutBf16;
        uint16_t* out = static_cast<uint16_t*>(p.out) + o;
        if (paired) {
          *reinterpret_cast<uint32_t*>(out) = bf16 ? pack_bf16(x0, x1) : pack_f16(x0, x1);
        } else {
          out[0] = mx_round16(x0, bf16);
          if (both) out[1] = mx_round16(x1, bf16);
        }
      }
    }
  }
}

template <int BN, bool GROUPED>
__global__ void __launch_bounds__(kMxFewThreads)
mx_few_kernel(const __grid_constant__ MxParams p) {
  using L = MxFewLayout<BN>;
  constexpr int STAGES = L::kStages;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~static_cast<uintptr_t>(1023));
  const uint32_t smem_base = smem_u32(smem);
  const uint32_t bar_base = smem_base + L::kBarOffset;
  const uint32_t bar_done = bar_base + 8u * (2 * STAGES), bar_retired = bar_done + 8u;
  uint32_t* tmem_holder = reinterpret_cast<uint32_t*>(smem + L::kMiscOffset);
  volatile int* s_abort = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 8);
  volatile int* s_tile = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 16);  // n0, m0, m_end, K blocks, x_col
  const AbortWord ab{s_abort, 0u};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int part = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / split;
  const int kb0 = static_cast<int>(static_cast<long long>(part) * p.num_kb / split);
  const int kb1 = static_cast<int>(static_cast<long long>(part + 1) * p.num_kb / split);

  auto load = [&](const MxTile& tl, int i, int stage) {  // K block i of this part
    const uint32_t bar = bar_base + 8u * stage, dst = smem_base + stage * L::kStageBytes;
    mbar_arrive_expect_tx(bar, L::kABytes + L::kBBytes + (GROUPED ? 2 : 4) * kMxSfBytes);
    tma_load_2d(dst, &p.tmap_w, bar, (kb0 + i) * kRowBytes, tl.w_row);
    tma_load_2d(dst + L::kABytes, &p.tmap_x, bar, (kb0 + i) * kRowBytes, tl.m0);
    tma_load_2d(dst + L::kSfOffset, &p.tmap_sw, bar, (kb0 + i) * 256, tl.w_block);
    if (!GROUPED) tma_load_2d(dst + L::kSfOffset + 2 * kMxSfBytes, &p.tmap_sx, bar, (kb0 + i) * 256, tl.x_block);
  };

  MxTile tl{0, 0, 0, 0, 0, 0, 0};
  int nkb = kb1 - kb0;
  if (!GROUPED && warp == 2 && elect_one()) {
    // The first weights start for the L2 before this launch's turn: a hint, and the L2 is where all writes meet, so that it
    // does no harm if the launch before is still making them. 1 x 4096 x 4096 back to back 4.6 us, 5.1 without; behind the
    // quantisation of x 6.4 and 6.75; 1 x 8192 x 8192 9.5 either way; twice as many blocks cost what they win. Grouped, where
    // the expert would have to be guessed, and in the tiled kernel it won less than 2%.
    const int n0 = tile % p.n_tiles * kBM;
    for (int i = 0; i < kMxFewAhead && i < nkb; ++i) {
      tma_prefetch_2d(&p.tmap_w, (kb0 + i) * kRowBytes, n0);
      tma_prefetch_2d(&p.tmap_sw, (kb0 + i) * 256, n0 >> 7);
    }
  }
  if (warp == 0) {
    if (elect_one()) {
      *s_abort = 0;
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(bar_base + 8u * s, GROUPED ? 2 : 1);  // the copies and, grouped, the scale warp
        mbar_init(bar_base + 8u * (STAGES + s), 1);
      }
      mbar_init(bar_done, 1);
      mbar_init(bar_retired, 1);
      mbar_init_fence();
      tma_prefetch_desc(&p.tmap_w);
      tma_prefetch_desc(&p.tmap_x);
      tma_prefetch_desc(&p.tmap_sw);
      if (!GROUPED) tma_prefetch_desc(&p.tmap_sx);
    }
    __syncwarp();
    pdl_wait();  // nothing before this line reads global memory (into the L2, at most)
    if (GROUPED) {
      if (!mx_few_tile<BN>(p, tile, lane, tl)) nkb = 0;
    } else {
      const int m_idx = tile / p.n_tiles;
      tl.n0 = tl.w_row = (tile - m_idx * p.n_tiles) * kBM;
      tl.w_block = tl.n0 >> 7;
      tl.m0 = m_idx * BN;
      tl.m_end = p.rows_x;
      tl.x_block = tl.m0 >> 7;
      tl.x_col = (tl.m0 & 127) >> 5;
    }
    if (elect_one()) {
      s_tile[0] = tl.n0;
      s_tile[1] = tl.m0;
      s_tile[2] = tl.m_end;
      s_tile[3] = nkb;
      s_tile[4] = tl.x_col;
      // the first copies need no one else: they fly while tensor memory is allocated and the CTA meets
      for (int i = 0; i < STAGES && i < nkb; ++i) load(tl, i, i);
    }
    __syncwarp();
  }
  if (warp == 1) {
    tmem_alloc(smem_u32(tmem_holder), L::kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem_base = *tmem_holder;
  tl.n0 = s_tile[0];
  tl.m0 = s_tile[1];
  tl.m_end = s_tile[2];
  nkb = s_tile[3];
  tl.x_col = s_tile[4];
  const int cnt = imin(BN, tl.m_end - tl.m0);
  pdl_wait();  // (returns at once: warp 0 has been through it)
  if (threadIdx.x == 0) pdl_trigger();
  if (GROUPED && nkb == 0) {  // no expert has this tile (all CTAs of the cluster see that)
    if (warp == 1) tmem_dealloc(tmem_base, L::kTmemCols);
    return;
  }

  if (warp == 0) {
    if (elect_one()) {
      int stage = 0;
      uint32_t phase = 0;
      int i = STAGES;
      for (; i < nkb; ++i) {
        if (!mbar_wait(bar_base + 8u * (STAGES + stage), phase, ab, kStatusTimeoutSmemEmpty, p.timeout_ns)) break;
        load(tl, i, stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (*s_abort != 0) {
        // give the copies in flight their time to land (1 ms per stage at most): none may outlive the CTA
        const AbortWord none{nullptr, 0u};
        for (int s = 0; s < STAGES && s < nkb; ++s)
          mbar_wait(bar_base + 8u * s, static_cast<uint32_t>(((i - 1 - s) / STAGES) & 1), none, 0, 1000000ull);
      }
    }
  } else if (warp == 1) {
    if (elect_one()) {
      const uint64_t a_desc0 = make_kmajor_sw128_desc(smem_base), b_desc0 = make_kmajor_sw128_desc(smem_base + L::kABytes);
      const uint64_t sf_desc0 = mx_sf_desc(smem_base + L::kSfOffset);
      int stage = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int i = 0; i < nkb; ++i) {
        if (!mbar_wait(bar_base + 8u * stage, phase, ab, kStatusTimeoutSmemFull, p.timeout_ns)) {
          ok = false;
          break;
        }
        tc_fence_after();
        const uint32_t off = static_cast<uint32_t>(stage) * (L::kStageBytes >> 4);
        // (a slot of scales per stage: it is free when the stage is)
        const uint32_t sf = tmem_base + BN + static_cast<uint32_t>(stage * L::kSfCols);
#pragma unroll
        for (int g = 0; g < 2; ++g)
#pragma unroll
          for (int b = 0; b < 2; ++b) mx_copy_sf<false>(sf + (g * 2 + b) * 4, sf_desc0 + off + static_cast<uint32_t>((b * 2 + g) * (kMxSfBytes >> 4)));
#pragma unroll
        for (int k = 0; k < 4; ++k) {
          const uint32_t sfa = sf + (k >> 1) * 8;
          umma_mxf4<false>(tmem_base, a_desc0 + off + 2u * k, b_desc0 + off + 2u * k, mx_idesc(128, BN, (k & 1) * 2), sfa, sfa + 4 + tl.x_col,
                           (i > 0 || k > 0) ? 1u : 0u);
        }
        umma_commit(bar_base + 8u * (STAGES + stage));
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
      if (ok) umma_commit(bar_done);
      if (*s_abort != 0) {  // UMMAs in flight still read shared memory and write tensor memory
        umma_commit(bar_retired);
        mbar_wait(bar_retired, 0, AbortWord{nullptr, 0u}, 0, 2000000ull);
      }
    }
  } else if (warp < 6) {
    // this CTA's accumulator, tokens x 128 output columns, into its shared memory (all loads have landed and all UMMAs
    // have retired by then, so the stages are free)
    const int quad = warp & 3;
    const int row = quad * 32 + lane;
    if (__all_sync(0xffffffffu, mbar_wait(bar_done, 0, ab, kStatusTimeoutTmemFull, p.timeout_ns))) {
      tc_fence_after();
      const uint32_t t0 = tmem_base + (static_cast<uint32_t>(quad * 32) << 16);
      constexpr int CH = BN < 32 ? BN : 32;
#pragma unroll 1
      for (int c = 0; c < BN && c < cnt; c += CH) {
        uint32_t r[CH];
        if constexpr (CH == 16) tmem_ld_32x16(t0 + c, r); else tmem_ld_32x32(t0 + c, r);
        tmem_ld_wait();
#pragma unroll
        for (int j = 0; j < CH; ++j) *reinterpret_cast<uint32_t*>(smem + ((c + j) * kBM + row) * 4) = r[j];
      }
      tc_fence_before();
    }
  } else if (GROUPED) {
    // the scales of the tile's tokens, four rows (lane, lane + 32, ...) and two groups of K a stage
    constexpr int UN = 4;  // stages whose loads are in flight together
    int stage = 0;
    uint32_t phase = 1;
    bool ok = true;
    for (int i0 = 0; ok && i0 < nkb; i0 += UN) {
      uint32_t w[UN][2][4];
#pragma unroll
      for (int u = 0; u < UN; ++u)
        if (i0 + u < nkb) mx_gather_scales<BN>(w[u], p, tl.m0, tl.m0 + cnt, kb0 + i0 + u, lane);
#pragma unroll
      for (int u = 0; u < UN; ++u) {
        if (i0 + u >= nkb || !ok) break;
        if (!__all_sync(0xffffffffu, mbar_wait(bar_base + 8u * (STAGES + stage), phase, ab, kStatusTimeoutSmemEmpty, p.timeout_ns))) {
          ok = false;
          break;
        }
        mx_put_scales(w[u], smem_base + stage * L::kStageBytes + L::kSfOffset + 2 * kMxSfBytes, lane);
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(bar_base + 8u * stage);
        if (++stage == STAGES) {
          stage = 0;
          phase ^= 1u;
        }
      }
    }
  }
  cluster_sync_all();
  if (warp >= 2 && warp < 6 && *s_abort == 0) {
    const int t = static_cast<int>(threadIdx.x) - 64;
    if (split == 1) mx_few_reduce<1, 8>(p, smem_base, tl, cnt, part, t);
    else if (split == 2) mx_few_reduce<2, 8>(p, smem_base, tl, cnt, part, t);
    else if (split == 4) mx_few_reduce<4, 8>(p, smem_base, tl, cnt, part, t);
    else mx_few_reduce<8, 4>(p, smem_base, tl, cnt, part, t);
  }
  cluster_sync_all();  // no CTA leaves while another still reads its shared memory
  if (*s_abort != 0 && threadIdx.x == 0) {
    *reinterpret_cast<volatile int*>(p.status) = *s_abort;
    __threadfence_system();
  }
  if (warp == 1) {
    tc_fence_after();
    tmem_dealloc(tmem_base, L::kTmemCols);
  }
}

}  // namespace fluxb
