// Host side of the microscaled 4-bit GEMMs (mx_gemm.cuh): checks, tensor maps, which kernel and tile a shape gets.
#include "internal.h"
#include "mx_gemm.cuh"

namespace fluxb {

template <class Kern>
static int mx_configure(Kern kern, int smem, bool* configured) {
  if (!*configured) {
    FLUXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    *configured = true;
  }
  return FLUXB_OK;
}

template <class Kern>
static int mx_launch(Kern kern, const MxParams& p, int grid, int threads, int smem, int cluster, bool early, cudaStream_t stream) {
  cudaLaunchConfig_t cfg;
  memset(&cfg, 0, sizeof(cfg));
  cfg.gridDim = dim3(grid, 1, 1);
  cfg.blockDim = dim3(threads, 1, 1);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = cluster;
  attr[0].val.clusterDim.y = 1;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = early ? 2 : 1;
  FLUXB_CUDA(cudaLaunchKernelEx(&cfg, kern, p));
  return FLUXB_OK;
}

template <int BN, bool CTA2, bool GROUPED>
static int launch_mx_tiles(const fluxb_comm* comm, const MxParams& p, long long most_tiles, int num_ctas, cudaStream_t stream) {
  using L = MxLayout<BN, CTA2, GROUPED>;
  auto kern = mx_gemm_kernel<BN, CTA2, GROUPED>;
  constexpr int smem = L::kTotal;
  static bool configured[64] = {};
  static int max_clusters[64] = {};
  const int dev = comm->device;
  FLUXB_REQUIRE(dev >= 0 && dev < 64, "device index %d not supported", dev);
  if (!configured[dev]) {
    FLUXB_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem));
    if (CTA2) {
      // how many CTA pairs can be resident at once: the persistent grid must not exceed it
      cudaLaunchConfig_t cfg;
      memset(&cfg, 0, sizeof(cfg));
      cfg.gridDim = dim3(comm->sm_count & ~1, 1, 1);
      cfg.blockDim = dim3(L::kThreads, 1, 1);
      cfg.dynamicSmemBytes = smem;
      cudaLaunchAttribute attr;
      attr.id = cudaLaunchAttributeClusterDimension;
      attr.val.clusterDim.x = 2;
      attr.val.clusterDim.y = 1;
      attr.val.clusterDim.z = 1;
      cfg.attrs = &attr;
      cfg.numAttrs = 1;
      int n = 0;
      FLUXB_CUDA(cudaOccupancyMaxActiveClusters(&n, kern, &cfg));
      FLUXB_REQUIRE(n >= 1, "no CTA pair of the 4-bit kernel fits on this device");
      max_clusters[dev] = n;
    }
    configured[dev] = true;
  }
  int workers = (num_ctas > 0 && num_ctas < comm->sm_count ? num_ctas : comm->sm_count) / (CTA2 ? 2 : 1);
  if (CTA2 && workers > max_clusters[dev]) workers = max_clusters[dev];
  if (workers > most_tiles) workers = static_cast<int>(most_tiles);
  if (workers < 1) workers = 1;
  return mx_launch(kern, p, workers * (CTA2 ? 2 : 1), L::kThreads, smem, CTA2 ? 2 : 1, comm->world == 1, stream);
}

template <int BN, bool GROUPED>
static int launch_mx_few(const fluxb_comm* comm, const MxParams& p, long long tiles, cudaStream_t stream) {
  auto kern = mx_few_kernel<BN, GROUPED>;
  static bool configured[64] = {};
  const int dev = comm->device;
  FLUXB_REQUIRE(dev >= 0 && dev < 64, "device index %d not supported", dev);
  const int rc = mx_configure(kern, MxFewLayout<BN>::kTotal, &configured[dev]);
  if (rc != FLUXB_OK) return rc;
  return mx_launch(kern, p, static_cast<int>(tiles * p.split), kMxFewThreads, MxFewLayout<BN>::kTotal, p.split, comm->world == 1, stream);
}

// Into how many parts along K the tiles of a few-token launch are cut: as many as keep all CTAs resident (two per SM up to
// 64 tokens, one above), with at least 2 K blocks each.
static int mx_few_split(int sm_count, long long tiles, int num_kb, int bn) {
  const long long slots = bn <= 64 ? 2 * sm_count : sm_count;
  int split = 1;
  while (split < kMxFewMaxSplit && 2 * split * tiles <= slots && num_kb / (2 * split) >= 2) split *= 2;
  return split;
}

static int mx_out_type(int out_dtype, int* ot) {
  switch (out_dtype) {
    case FLUXB_BF16: *ot = kOutBf16; return FLUXB_OK;
    case FLUXB_F16: *ot = kOutF16; return FLUXB_OK;
    case FLUXB_F32: *ot = kOutF32; return FLUXB_OK;
    default: FLUXB_FAIL(FLUXB_ERR_INVALID, "output dtype %d is not bf16/f16/f32", out_dtype);
  }
}

// Tiles of `bn` tokens that a grouped launch can need: an expert without tokens needs none, one with tokens at most one
// more than they fill.
static long long mx_most_tiles(int rows, int nexperts, int bn) { return static_cast<long long>(rows) / bn + (nexperts < rows ? nexperts : rows); }

// `per_group` = tokens that an expert gets on average (dense: all of them)
template <bool GROUPED>
static int mx_run(fluxb_comm* comm, MxParams& p, const void* xq, const void* wq, const void* ws, void* workspace, int k, int per_group,
                  const fluxb_tuning* tuning, cudaStream_t stream) {
  const int want_bn = tuning != nullptr ? tuning->block_n : 0, want_cg = tuning != nullptr ? tuning->cta_group : 0;
  const long long row_bytes = k / 2;
  const bool few = want_cg == 0 && (want_bn != 0 ? want_bn <= 128 : per_group <= 128);
  int bn = want_bn, cg = want_cg;
  if (few) {
    if (bn == 0) bn = per_group <= 16 ? 16 : per_group <= 32 ? 32 : per_group <= 64 ? 64 : 128;
    // the scales of a tile must start at an even column of tensor memory, that is at a multiple of 64 rows of a block
    // (an odd column raised a misaligned address); a grouped launch moves its tokens' scales to the tile's start
    FLUXB_REQUIRE(GROUPED || bn >= 64 || p.rows_x <= bn, "mx_gemm: block_n=%d is for up to %d tokens", bn, bn);
    cg = 1;
  } else {
    if (cg == 0) cg = 2;
    if (bn == 0) bn = 256;
  }
  const int tile_n = cg * kBM;
  const int groups = GROUPED ? p.nexperts : 1;
  p.n_tiles = (p.N + tile_n - 1) / tile_n;
  p.m_tiles = (p.rows_x + bn - 1) / bn;
  p.w_blocks = (p.N + 127) / 128;
  const long long tiles = (GROUPED ? mx_most_tiles(p.rows_x, groups, bn) : p.m_tiles) * p.n_tiles;
  FLUXB_REQUIRE(tiles < (1ll << 27), "mx_gemm: %d rows x %d columns have too many tiles", p.rows_x, p.N);
  p.band = tuning != nullptr && tuning->group_m > 0 ? tuning->group_m : 8;
  if (p.band > p.n_tiles) p.band = p.n_tiles;
  const long long words = static_cast<long long>(p.groups) * (kMxSfBytes / 4);
  int rc = encode_tmap_2d(&p.tmap_w, wq, FLUXB_S8, static_cast<long long>(groups) * p.N, row_bytes, row_bytes, kBM);
  if (rc != FLUXB_OK) return rc;
  rc = encode_tmap_2d(&p.tmap_x, xq, FLUXB_S8, p.rows_x, row_bytes, row_bytes, bn / cg);
  if (rc != FLUXB_OK) return rc;
  rc = encode_tmap_words(&p.tmap_sw, ws, static_cast<long long>(groups) * p.w_blocks, words, 1);
  if (rc != FLUXB_OK) return rc;
  const long long most_blocks = GROUPED ? mx_most_tiles(p.rows_x, groups, bn) * ((bn + 127) / 128) : 0;
  if (!GROUPED || cg == 2) {
    const void* blocks = GROUPED ? workspace : p.sx;
    rc = encode_tmap_words(&p.tmap_sx, blocks, GROUPED ? most_blocks : (p.rows_x + 127) / 128, words, (bn + 127) / 128);
    if (rc != FLUXB_OK) return rc;
  }
  if (few) {
    p.split = mx_few_split(comm->sm_count, GROUPED ? static_cast<long long>(groups) * p.n_tiles : tiles, p.num_kb, bn);
    switch (bn) {
      case 16: return launch_mx_few<16, GROUPED>(comm, p, tiles, stream);
      case 32: return launch_mx_few<32, GROUPED>(comm, p, tiles, stream);
      case 64: return launch_mx_few<64, GROUPED>(comm, p, tiles, stream);
      case 128: return launch_mx_few<128, GROUPED>(comm, p, tiles, stream);
      default: FLUXB_FAIL(FLUXB_ERR_INVALID, "mx_gemm: block_n=%d not in {16,32,64,128} for few tokens", bn);
    }
  }
  FLUXB_REQUIRE(cg == 2 ? bn == 64 || bn == 128 || bn == 192 || bn == 256 : cg == 1 && (bn == 64 || bn == 128),
                "mx_gemm: block_n=%d cta_group=%d is not {64,128} with 1 or {64,128,192,256} with 2", bn, cg);
  if (GROUPED && cg == 2) {
    const int parts = (p.groups + kMxRegroupGroups - 1) / kMxRegroupGroups;
    FLUXB_REQUIRE(most_blocks * parts < (1ll << 30), "mx_grouped_gemm: %d rows of %d groups are too many", p.rows_x, p.groups);
    rc = launch_pdl(mx_regroup_kernel, static_cast<int>(most_blocks * parts), kMxRegroupThreads, stream, p.sx, p.rows_x, p.groups, parts, bn, p.splits,
                    p.nexperts, static_cast<uint4*>(workspace));
    if (rc != FLUXB_OK) return rc;
  }
  const int num_ctas = tuning != nullptr ? tuning->num_ctas : 0;
  if (cg == 2) switch (bn) {
      case 64: return launch_mx_tiles<64, true, GROUPED>(comm, p, tiles, num_ctas, stream);
      case 128: return launch_mx_tiles<128, true, GROUPED>(comm, p, tiles, num_ctas, stream);
      case 192: return launch_mx_tiles<192, true, GROUPED>(comm, p, tiles, num_ctas, stream);
      default: return launch_mx_tiles<256, true, GROUPED>(comm, p, tiles, num_ctas, stream);
    }
  return bn == 64 ? launch_mx_tiles<64, false, GROUPED>(comm, p, tiles, num_ctas, stream) : launch_mx_tiles<128, false, GROUPED>(comm, p, tiles, num_ctas, stream);
}

static int mx_fill(const char* who, fluxb_comm* comm, MxParams& p, const void* xq, const void* xs, const void* wq, const void* ws, const void* out, int n, int k,
                   int out_dtype) {
  FLUXB_REQUIRE(comm != nullptr && xq != nullptr && xs != nullptr && wq != nullptr && ws != nullptr && out != nullptr, "%s: NULL argument", who);
  FLUXB_REQUIRE(k >= kMxBlock && k % kMxBlock == 0, "%s: k=%d must be a multiple of %d", who, k, kMxBlock);
  FLUXB_REQUIRE(n >= 1, "%s: n=%d invalid", who, n);
  FLUXB_REQUIRE(((reinterpret_cast<uintptr_t>(xq) | reinterpret_cast<uintptr_t>(xs) | reinterpret_cast<uintptr_t>(wq) | reinterpret_cast<uintptr_t>(ws)) & 15) == 0,
                "%s: operands and their scales must be 16-byte aligned", who);
  memset(&p, 0, sizeof(p));
  int rc = mx_out_type(out_dtype, &p.out_type);
  if (rc != FLUXB_OK) return rc;
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(out) & (p.out_type == kOutF32 ? 3 : 1)) == 0, "%s: the output is not aligned to its type", who);
  p.sx = static_cast<const uint8_t*>(xs);
  p.N = n;
  p.num_kb = (k + kMxStageK - 1) / kMxStageK;
  p.groups = (k + kMxGroupK - 1) / kMxGroupK;
  p.out = const_cast<void*>(out);
  p.ldo = n;
  p.out_blocks = p.out_type != kOutF32 && n % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15) == 0 ? 1 : 0;
  p.timeout_ns = comm->timeout_ns;
  p.status = comm->status_dev;
  return FLUXB_OK;
}

}  // namespace fluxb

using namespace fluxb;

extern "C" {

size_t fluxb_mx_scale_bytes(int batch, int rows, int k) {
  if (batch < 0 || rows < 0 || k < 0) return 0;
  return static_cast<size_t>(batch) * ((static_cast<size_t>(rows) + 127) / 128) * ((static_cast<size_t>(k) + kMxGroupK - 1) / kMxGroupK) * kMxSfBytes;
}

size_t fluxb_mx_grouped_workspace_bytes(int rows, int nexperts, int k) {
  if (rows < 0 || nexperts < 0 || k < 0) return 0;
  // the tile width that takes the most blocks: 64 (one for half as many rows), or 256 (two for an expert with one row)
  const long long most = mx_most_tiles(rows, nexperts, 64) + (nexperts < rows ? nexperts : rows);
  return static_cast<size_t>(most) * ((static_cast<size_t>(k) + kMxGroupK - 1) / kMxGroupK) * kMxSfBytes;
}

int fluxb_mx_gemm(fluxb_comm_t comm, const void* xq, const void* xs, const void* wq, const void* ws, void* out, int m, int n, int k, int out_dtype,
                  const void* bias, const fluxb_tuning* tuning, fluxb_stream_t stream) {
  FLUXB_REQUIRE(m >= 0, "mx_gemm: m=%d invalid", m);
  if (m == 0) return FLUXB_OK;
  MxParams p;
  const int rc = mx_fill("mx_gemm", comm, p, xq, xs, wq, ws, out, n, k, out_dtype);
  if (rc != FLUXB_OK) return rc;
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(bias) & (p.out_type == kOutF32 ? 3 : 1)) == 0, "mx_gemm: the bias is not aligned to its type");
  p.rows_x = m;
  p.bias = bias;
  return mx_run<false>(comm, p, xq, wq, ws, nullptr, k, m, tuning, static_cast<cudaStream_t>(stream));
}

int fluxb_mx_grouped_gemm(fluxb_comm_t comm, const void* xq, const void* xs, int rows, const void* wq, const void* ws, int nexperts,
                          const int* splits_dev, void* out, int n, int k, int out_dtype, void* workspace, const fluxb_tuning* tuning,
                          fluxb_stream_t stream) {
  FLUXB_REQUIRE(rows >= 0, "mx_grouped_gemm: rows=%d invalid", rows);
  FLUXB_REQUIRE(nexperts >= 1 && nexperts <= kMxMaxExperts, "mx_grouped_gemm: nexperts=%d out of [1,%d]", nexperts, kMxMaxExperts);
  if (rows == 0) return FLUXB_OK;
  FLUXB_REQUIRE(splits_dev != nullptr && workspace != nullptr, "mx_grouped_gemm: NULL argument");
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "mx_grouped_gemm: the workspace must be 16-byte aligned");
  FLUXB_REQUIRE(static_cast<long long>(nexperts) * n < (1ll << 31) - 256, "mx_grouped_gemm: %d experts of %d columns are too many", nexperts, n);
  MxParams p;
  const int rc = mx_fill("mx_grouped_gemm", comm, p, xq, xs, wq, ws, out, n, k, out_dtype);
  if (rc != FLUXB_OK) return rc;
  p.rows_x = rows;
  p.nexperts = nexperts;
  p.splits = splits_dev;
  const int used = nexperts < rows ? nexperts : rows;
  return mx_run<true>(comm, p, xq, wq, ws, workspace, k, (rows + used - 1) / used, tuning, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
