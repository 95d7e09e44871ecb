// Projections with bias, activation or gate, and residual in their epilogue: by streams of the weights for few rows
// (product_narrow.cuh), on CTA pairs for many (product_wide.cuh), by single loads where a row is not 16-byte aligned.
#include "product_narrow.cuh"
#include "product_wide.cuh"
#include "products.cuh"

namespace mie {
namespace {

int launch_any(const Product& p, cudaStream_t stream) {
  const int row_tiles = (p.m + kAnyTile - 1) / kAnyTile;
  MIE_CUDA(launch_chained(product_any_kernel<false>,
                          dim3((unsigned)((p.n + kAnyTile - 1) / kAnyTile), (unsigned)(row_tiles < 65535 ? row_tiles : 65535)),
                          dim3(128), 0, stream, p));
  MIE_LAUNCH_CHECK("product_any_kernel");
  return MIE_OK;
}

long long few_tiles(const Product& p) { return (p.n + (p.gated ? 63 : 127)) / (p.gated ? 64 : 128); }

// How many clusters of `parts` pairs the GPU runs at once.
int wide_clusters(int parts) {
  static int cached[64][8] = {{0}};
  int dev = 0;
  if (parts < 2 || parts > 7 || cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) return 0;
  if (cached[dev][parts] == 0) {
    int n = 0;
    cudaLaunchAttribute attr[2];
    cudaLaunchConfig_t config = wide_config<Rows::kDense, false, true>(attr, 1, parts, nullptr);
    config.numAttrs = 1;
    if (configure_wide<Rows::kDense, false, true>() != MIE_OK ||
        cudaOccupancyMaxActiveClusters(&n, product_wide_kernel<Rows::kDense, false, true>, &config) != cudaSuccess) {
      (void)cudaGetLastError();
      n = 0;
    }
    cached[dev][parts] = n > 0 ? n : -1;
  }
  return cached[dev][parts] > 0 ? cached[dev][parts] : 0;
}

// Clocks that a product takes: the choice between the kernels, and of their tiles.  The constants are fits to both kernels'
// times with every tile and cut, for 1 to 1024 rows of nine weights between 1000 x 1024 and 19456 x 2560 (gated): a fixed part
// (start, first loads, the last tile's epilogue, and what sums in parts cost), clocks of a block of 64 columns where a CTA or
// pair has its SMs' loads to itself and where all run, and all SMs' bytes a clock from HBM, which the weights come from once.
constexpr double kHbmBytes = 3400.0;

struct WidePlan {
  int rows, parts;  // of a tile; pairs that share its K
  double clocks;
};
WidePlan plan_wide(const Product& p) {
  const bool direct = direct_takes(p);
  const int channels = p.gated ? 128 : 256, pairs = sm_count() / 2, blocks = (p.k + 63) / 64;
  const long long weight_tiles = (p.n + channels - 1) / channels;
  WidePlan best = {0, 1, 0.0};
  const int most = p.m >= kWideRows ? kWideRows : p.m > 32 ? (p.m + 15) / 16 * 16 : 32;
  for (int rows = most; rows >= 32; rows -= 16) {
    const long long row_tiles = (p.m + rows - 1) / rows, tiles = weight_tiles * row_tiles;
    const double fresh = 32768.0 / (row_tiles < 8 ? row_tiles : 8) / kHbmBytes;
    const double few = 380.0 + 0.2 * rows > 2.36 * rows + 6.0 ? 380.0 + 0.2 * rows : 2.36 * rows + 6.0;
    const double all = 241.0 + 1.61 * rows > 390.0 ? 241.0 + 1.61 * rows : 390.0;
    const long long full = tiles / pairs, rest = tiles % pairs;
    double clocks = 10500.0 + full * blocks * (all > fresh * pairs ? all : fresh * pairs);
    const double last = 2 * rest > pairs && all > few ? all : few;
    if (rest > 0) clocks += blocks * (last > fresh * rest ? last : fresh * rest);
    if (best.rows == 0 || clocks < best.clocks) best = {rows, 1, clocks};
    for (int parts = 2; direct && parts <= 4 && blocks >= 4 * parts; parts *= 2) {
      if (tiles * parts > pairs || tiles > wide_clusters(parts)) break;
      const int own = (blocks + parts - 1) / parts;
      const double block = 2 * tiles * parts > pairs && all > few ? all : few, hbm = fresh * tiles * parts;
      const double fixed = parts == 2 ? 11500.0 + 0.13 * rows * rows : 13000.0 + 0.18 * rows * rows;
      const double time = fixed + own * (block > hbm ? block : hbm);
      if (time < best.clocks) best = {rows, parts, time};
    }
  }
  return best;
}
struct FewPlan {
  int rows, split;
  double clocks;
};
FewPlan plan_few(const Product& p) {
  const int blocks = (p.k + 63) / 64, sms = sm_count();
  FewPlan best = {0, 1, 0.0};
  for (int rows = 16; rows <= 128; rows *= 2) {
    const long long row_tiles = (p.m + rows - 1) / rows, tiles = few_tiles(p) * row_tiles;
    if (row_tiles > 8 && rows < 128) continue;
    if (rows > 16 && rows / 2 >= p.m) break;
    const int split = few_split(tiles, blocks, 2), own = (blocks + split - 1) / split;
    const double alone = rows == 16 ? 367.0 : rows == 32 ? 378.0 : rows == 64 ? 487.0 : 627.0;
    const double both = 2.0 * (16384.0 + 128.0 * rows) / 62.0;  // two CTAs on an SM
    const double fixed = rows == 16 ? 9500.0 : rows == 32 ? 11000.0 : rows == 64 ? 13500.0 : 16500.0;
    const double fresh = 16384.0 / row_tiles / kHbmBytes;
    const long long ctas = tiles * split, full = ctas / (2 * sms), rest = ctas % (2 * sms);
    double clocks = fixed + full * own * (both > fresh * 2 * sms ? both : fresh * 2 * sms);
    if (rest > 0) {
      const double last = rest <= sms ? alone : both;
      clocks += own * (last > fresh * rest ? last : fresh * rest);
    }
    if (best.rows == 0 || clocks < best.clocks) best = {rows, split, clocks};
  }
  return best;
}

int launch_dense_wide(const Product& p, const WidePlan& plan, cudaStream_t stream) {
  WideParams q = {};
  q.p = p;
  const int channels = p.gated ? 128 : 256;
  q.weight_tiles = (p.n + channels - 1) / channels;
  q.tile_rows = plan.rows;
  q.row_tiles = (p.m + q.tile_rows - 1) / q.tile_rows;
  q.band = 8;
  q.x_box = q.tile_rows / 2;
  WeightMaps maps;
  CUtensorMap map_x;
  const bool direct = direct_takes(p);
  if (int rc = weight_maps(&maps, p, 1, direct)) return rc;
  if (int rc = row_map(&map_x, p, p.m, q.x_box)) return rc;
  const long long tiles = (long long)q.row_tiles * q.weight_tiles;
  return p.gated  ? launch_wide<Rows::kDense, true, false>(maps, map_x, q, tiles, 1, stream)
         : direct ? launch_wide<Rows::kDense, false, true>(maps, map_x, q, tiles, plan.parts, stream)
                  : launch_wide<Rows::kDense, false, false>(maps, map_x, q, tiles, 1, stream);
}

template <int BN, bool kGated>
int launch_dense_few(const Product& p, int split, cudaStream_t stream) {
  FewParams q = {};
  q.p = p;
  CUtensorMap map_w, map_x;
  if (int rc = few_weight_map(&map_w, p, 1, kGated ? 64 : 128)) return rc;
  if (int rc = row_map(&map_x, p, p.m, BN)) return rc;
  return launch_few<BN, Few::kDense, kGated>(map_w, map_x, q, few_tiles(p), split, (p.m + BN - 1) / BN, stream);
}

template <bool kGated>
int launch_dense_few(const Product& p, const FewPlan& plan, cudaStream_t stream) {
  if (plan.rows == 16) return launch_dense_few<16, kGated>(p, plan.split, stream);
  if (plan.rows == 32) return launch_dense_few<32, kGated>(p, plan.split, stream);
  if (plan.rows == 64) return launch_dense_few<64, kGated>(p, plan.split, stream);
  return launch_dense_few<128, kGated>(p, plan.split, stream);
}

}  // namespace
}  // namespace mie

using namespace mie;

extern "C" int mie_fused_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                const void* residual, int64_t ldr, void* y, int64_t ldy, int32_t m, int32_t n, int32_t k,
                                int32_t activation, int32_t gated, int32_t* status, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  MIE_CHECK_ARG(x && w && y, "null pointer");
  MIE_CHECK_ARG(m >= 0 && n >= 1 && k >= 1 && m <= MIE_MAX_PRODUCT && n <= (1 << 30) && k <= MIE_MAX_PRODUCT,
                "invalid product %d x %d x %d", m, n, k);
  MIE_CHECK_ARG(ldx >= k && ldw >= k && ldy >= n && (!residual || ldr >= n), "a row is longer than its stride");
  MIE_CHECK_ARG(activation >= MIE_ACT_NONE && activation <= MIE_ACT_RELU, "unknown activation %d", activation);
  if (m == 0) return MIE_OK;
  Product p = {};
  p.x = (const __nv_bfloat16*)x, p.ldx = ldx;
  p.w = (const __nv_bfloat16*)w, p.ldw = ldw;
  p.bias = (const __nv_bfloat16*)bias;
  p.residual = (const __nv_bfloat16*)residual, p.ldr = ldr;
  p.y = y, p.ldy = ldy;
  p.m = m, p.n = n, p.k = k;
  p.activation = activation, p.gated = gated != 0, p.status = status;
  if (!wide_takes(p)) return launch_any(p, stream);
  const WidePlan wide = plan_wide(p);
  const FewPlan few = plan_few(p);
  // A grid has up to 65535 tiles of rows.
  if (wide.clocks < few.clocks || (m + few.rows - 1) / few.rows > 65535) return launch_dense_wide(p, wide, stream);
  return p.gated ? launch_dense_few<true>(p, few, stream) : launch_dense_few<false>(p, few, stream);
}
