// GEMMs of microscaled 4-bit operands (e2m1 values, one power of two for every 32 along K):
//   D[m, n] = sum over k of x[m, k] w[n, k] = sum over blocks b of 2^(sx[m, b] + sw[n, b] - 254) * sum of the block's products
// The tensor cores apply the scales (kind::mxf4, scale vectors 2X: 32 values); products of e2m1 values are exact, sums are
// in fp32.
//
// Operands are swapped as in the few-row GEMM: the 128 (or, for a CTA pair, 256) rows of a UMMA are rows of the weight,
// its N dimension is the tokens, 16 to 256 of them: a tile is as narrow as there are tokens, the weights of an expert
// with few tokens are not multiplied with padding, and a ragged end costs columns instead of 128-row boxes.
//
// A stage holds 256 values of K of every row of the tile: 128 bytes (swizzled, TMA) and 8 scale bytes. The scales stay
// row-major in memory ([rows, pitch] bytes), which any producer can write and any row offset can start at; the tensor
// cores want them in tensor memory, row r of a block of 128 in lane r % 32 of column r / 32, in all four quadrants.
// Loader warps (one per block of 128 rows) bring them: a lane reads its four rows' bytes and writes them as one 16-byte
// piece to shared memory, from where tcgen05.cp spreads 512 bytes (128 rows x 4 scales) at a time.
#pragma once
#include "gemm_kernel.cuh"

namespace fluxb {

constexpr int kMxBlock = 32;           // values that share a scale
constexpr int kMxStageK = 256;         // values of K per stage: 128 bytes
constexpr int kMxMaxExperts = 1024;
constexpr int kMxEpiWarps = 8;

struct MxParams {
  CUtensorMap tmap_w;  // weights [rows_w, K / 2 bytes]: 128 rows x 128 bytes
  CUtensorMap tmap_x;  // tokens [rows_x, K / 2 bytes]: this CTA's share of a tile's tokens x 128 bytes
  const uint8_t* sw;   // scales, `spw` / `spx` bytes a row (multiples of 16)
  const uint8_t* sx;
  long long spw, spx;
  int rows_w, rows_x;  // rows that exist: experts x N, tokens
  int N, num_kb, ksc;  // ksc = K / 32: scale bytes of a row that mean something
  int n_tiles, m_tiles, band;
  int nexperts;        // grouped: experts, else 0
  const int* splits;   // grouped: tokens per expert
  int out_type;
  void* out;
  long long ldo;
  const void* bias;    // [N] of the output's type, or null
  int split;           // few-token kernel: CTAs that share a tile's K
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

// Arrival that hands over shared memory written by this warp to the CTA of the pair that issues the UMMAs, and its wait.
__device__ __forceinline__ void mbar_arrive_release_cluster(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait_acquire_cluster(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred P;\n\t"
      "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 P, [%1], %2, %3;\n\t"
      "selp.u32 %0, 1, 0, P;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity), "r"(20000u)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ bool mbar_wait_acquire_cluster(uint32_t bar, uint32_t parity, const AbortWord& ab, int code, uint64_t budget_ns) {
  if (mbar_try_wait_acquire_cluster(bar, parity)) return true;
  const uint64_t t0 = globaltimer_ns();
  uint32_t n = 0;
  while (!mbar_try_wait_acquire_cluster(bar, parity)) {
    if ((++n & 31u) == 0u) {
      if (abort_seen(ab)) return false;
      if (globaltimer_ns() - t0 > budget_ns) {
        abort_raise(ab, code);
        return false;
      }
    }
  }
  return true;
}

template <int BN, bool CTA2>
struct MxLayout {
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBRows = CTA2 ? BN / 2 : BN;
  static constexpr int kBBytes = kBRows * kRowBytes;
  static constexpr int kSfBlocks = 1 + (BN + 127) / 128;  // blocks of 128 rows: the weights', the tokens' (all of them, in both CTAs of a pair)
  static constexpr int kSfOffset = kABytes + kBBytes;
  static constexpr int kStageBytes = kSfOffset + kSfBlocks * 1024;
  static constexpr int kStagesFit = (200 * 1024) / kStageBytes;
  static constexpr int kStages = kStagesFit > 8 ? 8 : kStagesFit;
  static constexpr int kSfCols = kSfBlocks * 8;  // tensor memory columns of a stage's scales
  static constexpr int kSlotsFit = (512 - 2 * BN) / kSfCols;
  static constexpr int kSlots = kSlotsFit > kStages ? kStages : kSlotsFit;
  static constexpr int kColsUsed = 2 * BN + kSlots * kSfCols;
  static constexpr uint32_t kTmemCols = kColsUsed <= 64 ? 64 : kColsUsed <= 128 ? 128 : kColsUsed <= 256 ? 256 : 512;
  static constexpr int kNumBars = 2 * kStages + 5;
  static constexpr int kBarOffset = kStages * kStageBytes;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kGroupOffset = kMiscOffset + 64;
  static constexpr int kGroupBytes = (2 * kMxMaxExperts + 2) * 4;
  static constexpr int total(bool grouped) { return kGroupOffset + (grouped ? kGroupBytes : 0) + 1024; }
  static constexpr int kThreads = 64 + 32 * kMxEpiWarps + 32 * kSfBlocks;
  static_assert(kStageBytes % 1024 == 0 && kSlots >= 2 && kStages >= 3, "layout");
};

// The groups of a grouped launch in shared memory: first row of every expert and the running number of token tiles, made
// by one warp. Splits that are negative or run past the rows that exist are cut, so that nothing outside is touched.
__device__ __forceinline__ void mx_group_table(const MxParams& p, int bn, int* row_first, int* tile_end, int lane) {
  long long rows = 0;
  int tiles = 0;
  for (int e0 = 0; e0 < p.nexperts; e0 += 32) {
    const int e = e0 + lane;
    long long m = e < p.nexperts ? p.splits[e] : 0;
    if (m < 0) m = 0;
    long long incl = m;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    long long first = rows + incl - m, end = rows + incl;
    if (first > p.rows_x) first = p.rows_x;
    if (end > p.rows_x) end = p.rows_x;
    const int mine = (static_cast<int>(end - first) + bn - 1) / bn;
    int tincl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tincl, off);
      if (lane >= off) tincl += v;
    }
    if (e < p.nexperts) {
      row_first[e] = static_cast<int>(first);
      tile_end[e] = tiles + tincl;
    }
    rows += __shfl_sync(0xffffffffu, incl, 31);
    tiles += __shfl_sync(0xffffffffu, tincl, 31);
    if (e0 + 32 >= p.nexperts && lane == 31) row_first[p.nexperts] = static_cast<int>(rows < p.rows_x ? rows : p.rows_x);
  }
}

// One output tile: rows [w_row, ...) of the weight matrix (n0 of its expert), tokens [m0, m_end).
struct MxTile {
  int n0, w_row, m0, m_end;
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
template <int BN, bool GROUPED>
__device__ __forceinline__ bool mx_tile(const MxParams& p, int tile_rows, int t, const int* row_first, const int* tile_end, MxTile& out) {
  int n_idx, m_idx;
  if (!GROUPED) {
    if (t >= p.n_tiles * p.m_tiles) return false;
    mx_raster(t, p.n_tiles, p.m_tiles, p.band, n_idx, m_idx);
    out.n0 = out.w_row = n_idx * tile_rows;
    out.m0 = m_idx * BN;
    out.m_end = p.rows_x;
    return true;
  }
  const int g = t / p.n_tiles;  // token tiles before this one, if all experts had whole ones: finds the expert
  int lo = 0, hi = p.nexperts;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (tile_end[mid] > g) hi = mid; else lo = mid + 1;
  }
  if (lo == p.nexperts) return false;
  const int before = lo > 0 ? tile_end[lo - 1] : 0;
  mx_raster(t - before * p.n_tiles, p.n_tiles, tile_end[lo] - before, p.band, n_idx, m_idx);
  out.n0 = n_idx * tile_rows;
  out.w_row = lo * p.N + out.n0;
  out.m0 = row_first[lo] + m_idx * BN;
  out.m_end = row_first[lo + 1];
  return true;
}

// The scales of four rows (first + lane, + 32, + 64, + 96) for one stage: 8 bytes each, zero for rows past `rows` and for
// bytes past the row's end (a scale of 255 there would make NaN of the zeros it meets).
struct MxScales {
  uint2 v[4];
};
__device__ __forceinline__ void mx_load_scales(MxScales& s, const uint8_t* base, long long pitch, int first, int rows, int kb, int ksc, int lane) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int r = first + q * 32 + lane;
    s.v[q] = r < rows ? __ldg(reinterpret_cast<const uint2*>(base + r * pitch + kb * 8)) : make_uint2(0u, 0u);
  }
  const int left = ksc - kb * 8;
  if (left < 8) {
    const uint32_t m0 = left >= 4 ? 0xFFFFFFFFu : left > 0 ? (1u << (8 * left)) - 1u : 0u;
    const uint32_t m1 = left > 4 ? (1u << (8 * (left - 4))) - 1u : 0u;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      s.v[q].x &= m0;
      s.v[q].y &= m1;
    }
  }
}
__device__ __forceinline__ void mx_store_scales(const MxScales& s, uint32_t dst, int lane) {
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + lane * 16), "r"(s.v[0].x), "r"(s.v[1].x), "r"(s.v[2].x), "r"(s.v[3].x) : "memory");
  asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(dst + 512 + lane * 16), "r"(s.v[0].y), "r"(s.v[1].y), "r"(s.v[2].y), "r"(s.v[3].y)
               : "memory");
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

// Persistent kernel. Warp 0: TMA; warp 1: tensor memory and UMMA; kMxEpiWarps epilogue warps, two per quadrant; then the
// loader warps of the scales. Two accumulators: the epilogue of a tile overlaps the main loop of the next.
template <int BN, bool CTA2, bool GROUPED>
__global__ void __launch_bounds__(MxLayout<BN, CTA2>::kThreads, 1)
mx_gemm_kernel(const __grid_constant__ MxParams p) {
  using L = MxLayout<BN, CTA2>;
  constexpr int STAGES = L::kStages, SLOTS = L::kSlots;
  constexpr int TILE_N = CTA2 ? 2 * kBM : kBM;
  static_assert(L::total(GROUPED) <= 232448, "shared memory budget exceeded");

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
  int* row_first = reinterpret_cast<int*>(smem + L::kGroupOffset);
  int* tile_end = row_first + kMxMaxExperts + 1;
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
      mbar_init(bar_full(s), 1 + (CTA2 ? 2 : 1) * L::kSfBlocks);  // the copies and the loader warps (of both CTAs)
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
    mx_group_table(p, BN, row_first, tile_end, lane);
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
      MxTile tl;
      for (int t = worker; ok && mx_tile<BN, GROUPED>(p, TILE_N, t, row_first, tile_end, tl); t += workers) {
        const int wrow = tl.w_row + half * kBM, xrow = tl.m0 + half * L::kBRows;
        for (int kb = 0; kb < p.num_kb; ++kb) {
          if (!mbar_wait(bar_empty(stage), phase ^ 1u, ab, kStatusTimeoutSmemEmpty, budget)) {
            ok = false;
            break;
          }
          if (arms) mbar_arrive_expect_tx(bar_full(stage), (CTA2 ? 2 : 1) * (L::kABytes + L::kBBytes));
          const uint32_t fb = full0 + 8u * stage;
          const uint32_t sa = smem_base + stage * L::kStageBytes;
          const int k = kb * kRowBytes;
          if (CTA2) {
            tma_load_2d_2cta(sa, &p.tmap_w, fb, k, wrow);
            tma_load_2d_2cta(sa + L::kABytes, &p.tmap_x, fb, k, xrow);
          } else {
            tma_load_2d(sa, &p.tmap_w, fb, k, wrow);
            tma_load_2d(sa + L::kABytes, &p.tmap_x, fb, k, xrow);
          }
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
      const uint32_t sf_tmem0 = tmem_base + 2 * BN;
      constexpr uint32_t UM = CTA2 ? 256 : 128;
      int stage = 0, slot = 0, it = 0, done = 0;  // `done` = stages issued so far, up to SLOTS
      uint32_t phase = 0;
      int old_stage = 0;                          // the stage that used this slot last, and its phase
      uint32_t old_phase = 0;
      bool ok = true;
      MxTile tl;
      for (int t = worker; ok && mx_tile<BN, GROUPED>(p, TILE_N, t, row_first, tile_end, tl); t += workers, ++it) {
        const int acc = it & 1;
        if (!mbar_wait<CTA2>(bar_tempty(acc), ((it >> 1) & 1) ^ 1u, ab, kStatusTimeoutTmemEmpty, budget)) break;
        tc_fence_after();
        const uint32_t d = tmem_base + static_cast<uint32_t>(acc * BN);
        for (int kb = 0; kb < p.num_kb; ++kb) {
          const bool full = CTA2 ? mbar_wait_acquire_cluster(bar_full(stage), phase, ab, kStatusTimeoutSmemFull, budget)
                                 : mbar_wait(bar_full(stage), phase, ab, kStatusTimeoutSmemFull, budget);
          if (!full) {
            ok = false;
            break;
          }
          // the scales' tensor memory is used again once the UMMAs that read it have retired
          if (SLOTS < STAGES) {
            if (done == SLOTS) {
              if (!mbar_wait(bar_empty(old_stage), old_phase, ab, kStatusTimeoutSmemEmpty, budget)) {
                ok = false;
                break;
              }
              if (++old_stage == STAGES) {
                old_stage = 0;
                old_phase ^= 1u;
              }
            } else {
              ++done;
            }
          }
          tc_fence_after();
          const uint32_t off = static_cast<uint32_t>(stage) * (L::kStageBytes >> 4);
          const uint32_t sf = sf_tmem0 + static_cast<uint32_t>(slot * L::kSfCols);
          // columns: per group of 128 values of K, 4 of the weights and 4 for every block of 128 tokens
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int b = 0; b < L::kSfBlocks; ++b)
              mx_copy_sf<CTA2>(sf + (g * L::kSfBlocks + b) * 4, sf_desc0 + off + static_cast<uint32_t>((b * 1024 + g * 512) >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t sfa = sf + (k >> 1) * L::kSfBlocks * 4;
            umma_mxf4<CTA2>(d, a_desc0 + off + 2u * k, b_desc0 + off + 2u * k, mx_idesc(UM, BN, (k & 1) * 2), sfa, sfa + 4, (kb > 0 || k > 0) ? 1u : 0u);
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
    constexpr int CH = BN < 32 ? BN : 32;
    int it = 0;
    MxTile tl;
    for (int t = worker; mx_tile<BN, GROUPED>(p, TILE_N, t, row_first, tile_end, tl); t += workers, ++it) {
      const int acc = it & 1;
      const int n = tl.n0 + half * kBM + quad * 32 + lane;
      const float bias = mx_bias(p, n);
      if (!__all_sync(0xffffffffu, mbar_wait(bar_tfull(acc), (it >> 1) & 1, ab, kStatusTimeoutTmemFull, budget, 100))) break;
      tc_fence_after();
      const uint32_t tacc = tmem_quad + static_cast<uint32_t>(acc * BN);
#pragma unroll 1
      for (int c = first * CH; c < BN && tl.m0 + c < tl.m_end; c += 2 * CH) {
        uint32_t r[CH];
        if constexpr (CH == 16) tmem_ld_32x16(tacc + c, r); else tmem_ld_32x32(tacc + c, r);
        tmem_ld_wait();
        mx_store_column<CH>(p, r, tl.m0 + c, tl.m_end - tl.m0 - c, n, bias);
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) {
        if (CTA2) mbar_arrive_cluster(tempty0 + 8u * acc); else mbar_arrive(tempty0 + 8u * acc);
      }
    }
  } else {
    // --------------------------------------------------------------- scales
    const int b = warp - 2 - kMxEpiWarps;  // block 0: the weights' rows of this CTA, then 128 tokens each
    const uint32_t full0 = CTA2 ? mapa_u32(bar_full(0), 0) : bar_full(0);
    const uint8_t* base = b == 0 ? p.sw : p.sx;
    const long long pitch = b == 0 ? p.spw : p.spx;
    const int rows_all = b == 0 ? p.rows_w : p.rows_x;
    constexpr int UN = 4;  // stages whose loads are in flight together
    int stage = 0;
    uint32_t phase = 0;
    bool ok = true;
    MxTile tl;
    for (int t = worker; ok && mx_tile<BN, GROUPED>(p, TILE_N, t, row_first, tile_end, tl); t += workers) {
      const int first = b == 0 ? tl.w_row + half * kBM : tl.m0 + (b - 1) * 128;
      const int rows = b == 0 ? rows_all : (rows_all < tl.m0 + BN ? rows_all : tl.m0 + BN);
      for (int kb0 = 0; ok && kb0 < p.num_kb; kb0 += UN) {
        MxScales s[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
          if (kb0 + u < p.num_kb) mx_load_scales(s[u], base, pitch, first, rows, kb0 + u, p.ksc, lane);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          if (kb0 + u >= p.num_kb || !ok) break;
          if (!__all_sync(0xffffffffu, mbar_wait(bar_empty(stage), phase ^ 1u, ab, kStatusTimeoutSmemEmpty, budget))) {
            ok = false;
            break;
          }
          mx_store_scales(s[u], smem_base + stage * L::kStageBytes + L::kSfOffset + b * 1024, lane);
          fence_proxy_async_smem();
          __syncwarp();
          if (lane == 0) {
            if (CTA2) mbar_arrive_release_cluster(full0 + 8u * stage); else mbar_arrive(full0 + 8u * stage);
          }
          if (++stage == STAGES) {
            stage = 0;
            phase ^= 1u;
          }
        }
      }
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

// ------------------------------------------------------------------------------------------------------- few tokens
// Few tokens (up to 128, or a few per expert), where the time is that of reading the weights once and of getting started:
// one output tile per cluster of `split` CTAs, which cut K. Each CTA leaves its accumulator in its own shared memory; after
// a cluster barrier CTA r sums the tokens r * per ... of all parts, in rank order, through distributed shared memory: no
// scratch, no counters, any number of launches side by side. A grouped launch has a cluster for every tile that the
// experts could need (the counts are on the device); those that no expert needs leave at once.
constexpr int kMxFewThreads = 256;  // warp 0 TMA, warp 1 UMMA + tensor memory, warps 2-5 read-out and output, 6-7 scales
constexpr int kMxFewMaxSplit = 8;

template <int BN>
struct MxFewLayout {
  static constexpr int kABytes = kBM * kRowBytes;
  static constexpr int kBBytes = BN * kRowBytes;
  static constexpr int kSfOffset = kABytes + kBBytes;
  static constexpr int kStageBytes = kSfOffset + 2048;
  // up to 64 tokens a CTA takes half of an SM's shared memory, so that one CTA's prologue and reduction overlap another's loads
  static constexpr int kStages = BN == 16 ? 5 : BN <= 64 ? 4 : 6;
  static_assert(BN <= 128 && kStages * kStageBytes >= BN * kBM * 4, "the read-out must fit into the stages");
  static constexpr int kSfCols = 16;
  static constexpr int kColsUsed = BN + kStages * kSfCols;
  static constexpr uint32_t kTmemCols = kColsUsed <= 128 ? 128 : 256;
  static constexpr int kNumBars = 2 * kStages + 2;  // full / empty per stage, accumulator complete, "UMMAs retired" (abort path)
  static constexpr int kBarOffset = kStages * kStageBytes;
  static constexpr int kMiscOffset = kBarOffset + kNumBars * 8;
  static constexpr int kTotal = kMiscOffset + 64 + 1024;  // + slack for 1024-byte alignment
};

// The tile of cluster `t` of a grouped launch, by one warp: the expert whose token tiles hold it. False: no expert has it.
template <int BN>
__device__ __forceinline__ bool mx_few_tile(const MxParams& p, int t, int lane, MxTile& out) {
  const int g = t / p.n_tiles;
  long long rows = 0;
  int tiles = 0;
  for (int e0 = 0; e0 < p.nexperts; e0 += 32) {
    const int e = e0 + lane;
    long long m = e < p.nexperts ? p.splits[e] : 0;
    if (m < 0) m = 0;
    long long incl = m;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const long long v = __shfl_up_sync(0xffffffffu, incl, off);
      if (lane >= off) incl += v;
    }
    long long first = rows + incl - m, end = rows + incl;
    if (first > p.rows_x) first = p.rows_x;
    if (end > p.rows_x) end = p.rows_x;
    const int mine = (static_cast<int>(end - first) + BN - 1) / BN;
    int tincl = mine;
#pragma unroll
    for (int off = 1; off < 32; off <<= 1) {
      const int v = __shfl_up_sync(0xffffffffu, tincl, off);
      if (lane >= off) tincl += v;
    }
    const unsigned has = __ballot_sync(0xffffffffu, tiles + tincl > g);
    if (has != 0) {
      const int src = __ffs(has) - 1;
      const int f = __shfl_sync(0xffffffffu, static_cast<int>(first), src);
      const int before = __shfl_sync(0xffffffffu, tiles + tincl - mine, src);
      out.m_end = __shfl_sync(0xffffffffu, static_cast<int>(end), src);
      const int n_idx = (t - before * p.n_tiles) % p.n_tiles, m_idx = g - before;
      out.n0 = n_idx * kBM;
      out.w_row = (e0 + src) * p.N + out.n0;
      out.m0 = f + m_idx * BN;
      return true;
    }
    rows += __shfl_sync(0xffffffffu, incl, 31);
    tiles += __shfl_sync(0xffffffffu, tincl, 31);
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
  volatile int* s_tile = reinterpret_cast<volatile int*>(smem + L::kMiscOffset + 16);  // n0, w_row, m0, m_end, K blocks
  const AbortWord ab{s_abort, 0u};
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int split = p.split;
  const int part = static_cast<int>(cluster_ctarank());
  const int tile = static_cast<int>(blockIdx.x) / split;
  const int kb0 = static_cast<int>(static_cast<long long>(part) * p.num_kb / split);
  const int kb1 = static_cast<int>(static_cast<long long>(part + 1) * p.num_kb / split);

  auto load = [&](const MxTile& tl, int i, int stage) {  // K block i of this part
    const uint32_t bar = bar_base + 8u * stage, dst = smem_base + stage * L::kStageBytes;
    const int k = (kb0 + i) * kRowBytes;
    mbar_arrive_expect_tx(bar, L::kABytes + L::kBBytes);
    tma_load_2d(dst, &p.tmap_w, bar, k, tl.w_row);
    tma_load_2d(dst + L::kABytes, &p.tmap_x, bar, k, tl.m0);
  };

  MxTile tl{0, 0, 0, 0};
  int nkb = kb1 - kb0;
  if (warp == 0) {
    if (elect_one()) {
      *s_abort = 0;
      for (int s = 0; s < STAGES; ++s) {
        mbar_init(bar_base + 8u * s, 3);  // the copies and the two loader warps
        mbar_init(bar_base + 8u * (STAGES + s), 1);
      }
      mbar_init(bar_done, 1);
      mbar_init(bar_retired, 1);
      mbar_init_fence();
    }
    __syncwarp();
    pdl_wait();  // nothing before this line reads global memory
    if (GROUPED) {
      if (!mx_few_tile<BN>(p, tile, lane, tl)) nkb = 0;
    } else {
      const int m_idx = tile / p.n_tiles;
      tl.n0 = tl.w_row = (tile - m_idx * p.n_tiles) * kBM;
      tl.m0 = m_idx * BN;
      tl.m_end = p.rows_x;
    }
    if (elect_one()) {
      s_tile[0] = tl.n0;
      s_tile[1] = tl.w_row;
      s_tile[2] = tl.m0;
      s_tile[3] = tl.m_end;
      s_tile[4] = nkb;
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
  tl.w_row = s_tile[1];
  tl.m0 = s_tile[2];
  tl.m_end = s_tile[3];
  nkb = s_tile[4];
  const int cnt = nkb == 0 ? 0 : imin(BN, tl.m_end - tl.m0);
  pdl_wait();  // (returns at once: warp 0 has been through it)
  if (threadIdx.x == 0) pdl_trigger();

  if (nkb > 0) {
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
          const uint32_t sf = tmem_base + BN + static_cast<uint32_t>(stage * L::kSfCols);
#pragma unroll
          for (int g = 0; g < 2; ++g)
#pragma unroll
            for (int b = 0; b < 2; ++b) mx_copy_sf<false>(sf + (g * 2 + b) * 4, sf_desc0 + off + static_cast<uint32_t>((b * 1024 + g * 512) >> 4));
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            const uint32_t sfa = sf + (k >> 1) * 8;
            umma_mxf4<false>(tmem_base, a_desc0 + off + 2u * k, b_desc0 + off + 2u * k, mx_idesc(128, BN, (k & 1) * 2), sfa, sfa + 4,
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
    } else {
      const bool weights = warp == 6;
      const int first = weights ? tl.w_row : tl.m0, rows = weights ? p.rows_w : tl.m0 + cnt;
      constexpr int UN = 4;  // stages whose loads are in flight together
      int stage = 0;
      uint32_t phase = 1;
      bool ok = true;
      for (int i0 = 0; ok && i0 < nkb; i0 += UN) {
        MxScales s[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u)
          if (i0 + u < nkb) mx_load_scales(s[u], weights ? p.sw : p.sx, weights ? p.spw : p.spx, first, rows, kb0 + i0 + u, p.ksc, lane);
#pragma unroll
        for (int u = 0; u < UN; ++u) {
          if (i0 + u >= nkb || !ok) break;
          if (!__all_sync(0xffffffffu, mbar_wait(bar_base + 8u * (STAGES + stage), phase, ab, kStatusTimeoutSmemEmpty, p.timeout_ns))) {
            ok = false;
            break;
          }
          mx_store_scales(s[u], smem_base + stage * L::kStageBytes + L::kSfOffset + (weights ? 0 : 1024), lane);
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
  }
  cluster_sync_all();
  if (warp >= 2 && warp < 6 && cnt > 0 && *s_abort == 0) {
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
