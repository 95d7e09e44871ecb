// Projections with bias, activation or gate, and residual in their epilogue.
#include "product_narrow.cuh"
#include "product_wide.cuh"
#include "products.cuh"

namespace mie {
namespace {

constexpr int kFewRows = 128;

int launch_any(const Product& p, cudaStream_t stream) {
  const int row_tiles = (p.m + kAnyTile - 1) / kAnyTile;
  MIE_CUDA(launch_chained(product_any_kernel<false>,
                          dim3((unsigned)((p.n + kAnyTile - 1) / kAnyTile), (unsigned)(row_tiles < 65535 ? row_tiles : 65535)),
                          dim3(128), 0, stream, p));
  MIE_LAUNCH_CHECK("product_any_kernel");
  return MIE_OK;
}

int launch_dense_wide(const Product& p, cudaStream_t stream) {
  WideParams q = {};
  q.p = p;
  const int channels = p.gated ? 128 : 256, pairs = sm_count() / 2;
  q.weight_tiles = (p.n + channels - 1) / channels;
  // Rows of a tile: the time is the rounds' number times the rows, below 128 of which the weights' way through shared memory
  // takes as long.
  long long best = 0;
  for (int rows = kWideRows; rows >= 128; rows -= 16) {
    const long long tiles = (long long)q.weight_tiles * ((p.m + rows - 1) / rows);
    const long long cost = (tiles + pairs - 1) / pairs * (rows + 16);
    if (q.tile_rows == 0 || cost < best) {
      best = cost;
      q.tile_rows = rows;
    }
  }
  q.row_tiles = (p.m + q.tile_rows - 1) / q.tile_rows;
  q.band = 8;
  q.x_box = q.tile_rows / 2;
  WeightMaps maps;
  CUtensorMap map_x;
  const bool direct = direct_takes(p);
  if (int rc = weight_maps(&maps, p, 1, direct)) return rc;
  if (int rc = row_map(&map_x, p, p.m, q.x_box)) return rc;
  const long long tiles = (long long)q.row_tiles * q.weight_tiles;
  return p.gated  ? launch_wide<Rows::kDense, true, false>(maps, map_x, q, tiles, stream)
         : direct ? launch_wide<Rows::kDense, false, true>(maps, map_x, q, tiles, stream)
                  : launch_wide<Rows::kDense, false, false>(maps, map_x, q, tiles, stream);
}

template <int BN, bool kGated>
int launch_dense_few(const Product& p, cudaStream_t stream) {
  FewParams q = {};
  q.p = p;
  const long long tiles = (p.n + (kGated ? 63 : 127)) / (kGated ? 64 : 128);
  CUtensorMap map_w, map_x;
  if (int rc = few_weight_map(&map_w, p, 1)) return rc;
  if (int rc = row_map(&map_x, p, p.m, BN)) return rc;
  return launch_few<BN, Few::kDense, kGated>(map_w, map_x, q, tiles,
                                             few_split(tiles, (p.k + 63) / 64, FewSmem<BN, Few::kDense>::kCtasPerSm), stream);
}

template <bool kGated>
int launch_dense_few(const Product& p, cudaStream_t stream) {
  if (p.m <= 16) return launch_dense_few<16, kGated>(p, stream);
  if (p.m <= 32) return launch_dense_few<32, kGated>(p, stream);
  if (p.m <= 64) return launch_dense_few<64, kGated>(p, stream);
  return launch_dense_few<128, kGated>(p, stream);
}

}  // namespace
}  // namespace mie

using namespace mie;

extern "C" int mie_fused_linear(const void* x, int64_t ldx, const void* w, int64_t ldw, const void* bias,
                                const void* residual, int64_t ldr, void* y, int64_t ldy, int32_t m, int32_t n, int32_t k,
                                int32_t activation, int32_t gated, int32_t* status, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  MIE_CHECK_ARG(x && w && y, "null pointer");
  MIE_CHECK_ARG(m >= 0 && n >= 1 && k >= 1 && n <= (1 << 30), "invalid product %d x %d x %d", m, n, k);
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
  if (m <= kFewRows) return p.gated ? launch_dense_few<true>(p, stream) : launch_dense_few<false>(p, stream);
  return launch_dense_wide(p, stream);
}
