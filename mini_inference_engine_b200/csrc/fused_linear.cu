// Projections with bias, activation or gate, and residual in their epilogue.
#include "products.cuh"

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
  const int row_tiles = (m + kAnyTile - 1) / kAnyTile;
  MIE_CUDA(launch_chained(product_any_kernel<false>,
                          dim3((unsigned)((n + kAnyTile - 1) / kAnyTile), (unsigned)(row_tiles < 65535 ? row_tiles : 65535)),
                          dim3(128), 0, stream, p));
  MIE_LAUNCH_CHECK("product_any_kernel");
  return MIE_OK;
}
