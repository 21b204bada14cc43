// Host side of the microscaled 4-bit GEMMs (mx_gemm.cuh): checks, tensor maps, which kernel and tile a shape gets.
#include <math.h>

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

// Which kernel and tile a launch gets: the one whose time, estimated from what it has to do, is the shortest. The estimates
// are linear in the launch's numbers, with coefficients (us) fitted to measured times of all variants on 148 problems
// (dense 1 .. 4096 x 1024 .. 28672 x 1024 .. 8192; 8 to 128 experts, 2 to 65536 rows, of 1024 .. 14336 x 1024 .. 8192;
// weights from memory, launches back to back in a graph). Over those problems the choice takes 2% longer than the fastest
// variant on average, 24% at worst (64 x 4096 x 4096 6.7 us against 5.4, grouped 11%). Over 297 others, down to 512 x 416, it is 3%
// on average and, by how long the launch takes, at worst: up to 10 us 42% (64 x 1000 x 416 5.4 us against 3.8), up to 20 us 10%, up to
// 40 us 8%, beyond 6% (dense) and 17% (grouped). The last is a K longer than any that was fitted: 8 experts x 4096 x 14336 with 16 and
// 64 tokens, top-2, 50.4 and 52.6 us, where the few-token kernel's 64 tokens uncut take 43.6 and 45.1; 8192 tokens over 64 experts take
// 8 to 9% longer in tiles of 192 than of 256. One variant for all would be far off on either side: 256 x 4096 x 4096 takes 5.9 us in
// tiles of 64 and 9.7 in tiles of 256, 4096 x 8192 x 8192 160 and 90.
//   tiled:      fixed + waves * (per_stage * K blocks + per_wave) + per_mb * MB of weights (+ grouped)
//   few tokens: fixed + per_stage * K blocks of a part + per_cta * CTAs per slot + per_block * K blocks per slot
//               + per_mb * MB of weights (+ grouped)
struct MxTileCost {
  int bn, cg;
  float fixed, per_stage, per_wave, per_mb, grouped;
};
constexpr MxTileCost kMxTileCosts[] = {
    {64, 1, 1.58f, 0.142f, 0.712f, 0.1007f, 2.83f},  {128, 1, 1.33f, 0.191f, 1.159f, 0.0981f, 3.77f}, {64, 2, 2.32f, 0.121f, 0.609f, 0.0989f, 5.35f},
    {128, 2, 2.43f, 0.153f, 0.918f, 0.0844f, 4.94f}, {192, 2, 2.46f, 0.222f, 1.131f, 0.0729f, 5.13f}, {256, 2, 3.05f, 0.293f, 1.160f, 0.0543f, 4.71f},
};
struct MxFewCost {
  int bn;
  float fixed, per_stage, per_cta, per_block, per_mb, grouped;
};
constexpr MxFewCost kMxFewCosts[] = {
    {16, 0.87f, 0.216f, 5.49f, 0.147f, 0.079f, 0.26f}, {32, 0.79f, 0.249f, 5.61f, 0.073f, 0.099f, 0.24f}, {64, 1.06f, 0.260f, 5.78f, 0.031f, 0.110f, 0.11f},
};
struct MxChoice {
  int bn = 0, cg = 0, split = 0;  // split > 0: the few-token kernel
};
// `nexperts` 0: dense. `want_bn`, `want_cg`: the caller's choice of a kernel and tile, 0 = none.
static MxChoice mx_choose(int sm_count, int nexperts, int rows, int n, int num_kb, double weight_mb, int want_bn, int want_cg) {
  double used = 1.0, per = rows, longest = rows;
  if (nexperts > 0) {
    // experts that get rows if every row falls on one at random, and a good guess at what the longer of them get
    used = nexperts > 1 ? nexperts * (1.0 - exp(rows * log1p(-1.0 / nexperts))) : 1.0;
    per = rows / used;
    longest = per + sqrt(per);
  }
  auto token_tiles = [&](int bn) {
    if (nexperts == 0) return ceil(static_cast<double>(rows) / bn);
    return longest <= 4.0 * bn ? used * ceil(longest / bn) : used * (per / bn + 0.5);
  };
  const double mb = used * weight_mb, grouped = nexperts > 0 ? 1.0 : 0.0;
  MxChoice best;
  double least = 0.0;
  auto offer = [&](double us, int bn, int cg, int split) {
    if (best.bn != 0 && us >= least) return;
    best.bn = bn;
    best.cg = cg;
    best.split = split;
    least = us;
  };
  for (const MxTileCost& c : kMxTileCosts) {
    if ((want_bn != 0 || want_cg != 0) && (c.cg != want_cg || (want_bn != 0 && c.bn != want_bn))) continue;
    const double tiles = token_tiles(c.bn) * ((n + kBM * c.cg - 1) / (kBM * c.cg));
    const double waves = ceil(tiles / (sm_count / c.cg) - 1e-9);
    offer(c.fixed + waves * (c.per_stage * num_kb + c.per_wave) + c.per_mb * mb + c.grouped * grouped, c.bn, c.cg, 0);
  }
  for (const MxFewCost& c : kMxFewCosts) {
    if (want_cg != 0 || (want_bn != 0 ? c.bn != want_bn : per > 96)) continue;
    if (nexperts == 0 && c.bn < 64 && rows > c.bn) continue;  // (see mx_run)
    const double tiles = token_tiles(c.bn) * ((n + kBM - 1) / kBM);
    for (int split = 1; split <= kMxFewMaxSplit && split <= num_kb; split *= 2)
      offer(c.fixed + c.per_stage * num_kb / split + c.per_cta * tiles * split / (2 * sm_count) + c.per_block * tiles * num_kb / (2 * sm_count) + c.per_mb * mb +
                c.grouped * grouped,
            c.bn, 1, split);
  }
  return best;
}

// A tile's last row is a 31-bit integer, too.
constexpr int kMxMostRows = 0x7FFFFFFF - 512;

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

template <bool GROUPED>
static int mx_run(fluxb_comm* comm, MxParams& p, const void* xq, const void* wq, const void* ws, void* workspace, int k, const fluxb_tuning* tuning,
                  cudaStream_t stream) {
  const int want_bn = tuning != nullptr ? tuning->block_n : 0, want_cg = tuning != nullptr ? tuning->cta_group : 0;
  const long long row_bytes = k / 2;
  // the scales of a tile must start at an even column of tensor memory, that is at a multiple of 64 rows of a block (an odd
  // column raised a misaligned address); a grouped launch moves its tokens' scales to the tile's start
  FLUXB_REQUIRE(GROUPED || want_cg != 0 || want_bn == 0 || want_bn >= 64 || p.rows_x <= want_bn, "mx_gemm: block_n=%d is for up to %d tokens", want_bn,
                want_bn);
  const MxChoice choice = mx_choose(comm->sm_count, p.nexperts, p.rows_x, p.N, p.num_kb, p.N * (row_bytes + k / kMxBlock) * 1e-6, want_bn, want_cg);
  FLUXB_REQUIRE(choice.bn != 0, "mx_gemm: block_n=%d cta_group=%d is not {16,32,64} with 0, {64,128} with 1 or {64,128,192,256} with 2", want_bn, want_cg);
  const int bn = choice.bn, cg = choice.cg;
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
  p.split = choice.split;
  if (p.split > 0) {
    if (bn == 16) return launch_mx_few<16, GROUPED>(comm, p, tiles, stream);
    if (bn == 32) return launch_mx_few<32, GROUPED>(comm, p, tiles, stream);
    return launch_mx_few<64, GROUPED>(comm, p, tiles, stream);
  }
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
  FLUXB_REQUIRE(n >= 1 && n <= kMxMostRows, "%s: n=%d invalid", who, n);
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
  FLUXB_REQUIRE(comm->ranks_on_gpu <= 1, "%s: not while several ranks share the GPU", who);  // (calls only queue their work then)
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
  FLUXB_REQUIRE(m >= 0 && m <= kMxMostRows, "mx_gemm: m=%d invalid", m);
  if (m == 0) return FLUXB_OK;
  MxParams p;
  const int rc = mx_fill("mx_gemm", comm, p, xq, xs, wq, ws, out, n, k, out_dtype);
  if (rc != FLUXB_OK) return rc;
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(bias) & (p.out_type == kOutF32 ? 3 : 1)) == 0, "mx_gemm: the bias is not aligned to its type");
  p.rows_x = m;
  p.bias = bias;
  return mx_run<false>(comm, p, xq, wq, ws, nullptr, k, tuning, static_cast<cudaStream_t>(stream));
}

int fluxb_mx_grouped_gemm(fluxb_comm_t comm, const void* xq, const void* xs, int rows, const void* wq, const void* ws, int nexperts,
                          const int* splits_dev, void* out, int n, int k, int out_dtype, void* workspace, const fluxb_tuning* tuning,
                          fluxb_stream_t stream) {
  FLUXB_REQUIRE(rows >= 0 && rows <= kMxMostRows, "mx_grouped_gemm: rows=%d invalid", rows);
  FLUXB_REQUIRE(nexperts >= 1 && nexperts <= kMxMaxExperts, "mx_grouped_gemm: nexperts=%d out of [1,%d]", nexperts, kMxMaxExperts);
  if (rows == 0) return FLUXB_OK;
  FLUXB_REQUIRE(splits_dev != nullptr && workspace != nullptr, "mx_grouped_gemm: NULL argument");
  FLUXB_REQUIRE((reinterpret_cast<uintptr_t>(workspace) & 15) == 0, "mx_grouped_gemm: the workspace must be 16-byte aligned");
  FLUXB_REQUIRE(all_aligned(4, {splits_dev}), "mx_grouped_gemm: splits must be aligned to their type");
  FLUXB_REQUIRE(static_cast<long long>(nexperts) * n < (1ll << 31) - 256, "mx_grouped_gemm: %d experts of %d columns are too many", nexperts, n);
  MxParams p;
  const int rc = mx_fill("mx_grouped_gemm", comm, p, xq, xs, wq, ws, out, n, k, out_dtype);
  if (rc != FLUXB_OK) return rc;
  p.rows_x = rows;
  p.nexperts = nexperts;
  p.splits = splits_dev;
  return mx_run<true>(comm, p, xq, wq, ws, workspace, k, tuning, static_cast<cudaStream_t>(stream));
}

}  // extern "C"
