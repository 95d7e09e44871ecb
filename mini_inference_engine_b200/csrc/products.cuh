// Products of bf16 rows with weight rows, finished in their epilogue:
//
//   y[r] = act(x[r] W^T + b) + res[r],   gated, W = [G; U]:  y[r] = act(x[r] G^T + b_g) * (x[r] U^T + b_u) + res[r]
//
// over one weight (fused_linear.cu) or over one weight per expert, with rows sorted by expert (expert_mlp.cu).
#pragma once

#include "common.cuh"
#include "glue.cuh"

namespace mie {

// Rows of one expert: sorted rows [first, first + count).
struct RowTile {
  int expert, first, count, unused;
};

struct Product {
  const __nv_bfloat16* x;
  long long ldx;
  const __nv_bfloat16* w;
  long long ldw, w_expert;  // strides of a weight row and of an expert
  const __nv_bfloat16* bias;
  const __nv_bfloat16* residual;
  long long ldr;
  void* y;  // bf16, or fp32 (`wide`)
  long long ldy;
  int m, n, k;  // rows, columns of y, length of the sums; a gated weight has 2 n rows
  int activation, gated, wide;
  // Over experts: the tiles, how many there are, and for a sorted row the row of x that it reads (source, divided by
  // source_divisor; its own without one) and its factor (by source).
  const RowTile* tiles;
  const int* tile_count;
  const int* source;
  int source_divisor;
  const float* factor;
  int* status;
};

namespace {

__device__ __forceinline__ float activate(int kind, float z) {
  if (kind == MIE_ACT_SILU) {
    const float d = gate_denominator(z * -kLog2e);
    return d > kGateLimit ? gate_sigmoid(z) : gate_quotient(z, d);
  }
  if (kind == MIE_ACT_GELU) {
    const float inner = 0.7978845608028654f * (z + 0.044715f * z * z * z);
    const float d = gate_denominator(inner * (-2.f * kLog2e));
    return d > kGateLimit ? -0.f * (z * 0.f + 1.f) : gate_quotient(z, d);
  }
  if (kind == MIE_ACT_RELU) return z > 0.f || z != z ? z : 0.f;
  return z;
}

// The activation of N values at once: their exponentials and reciprocals overlap, and one test finds the thread that has a
// value whose reciprocal would be flushed (value by value the branches cost 190 clocks each in the pair kernel's epilogue).
template <int N>
__device__ __forceinline__ void activate_all(int kind, float (&z)[N]) {
  if (kind == MIE_ACT_SILU || kind == MIE_ACT_GELU) {
    float d[N], top = 0.f;  // NaN passes the test and comes through the quotient
    if (kind == MIE_ACT_SILU) {
#pragma unroll
      for (int i = 0; i < N; ++i) d[i] = gate_denominator(z[i] * -kLog2e);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i)
        d[i] = gate_denominator(z[i] * fmaf(z[i] * z[i], -2.f * kLog2e * 0.7978845608028654f * 0.044715f,
                                            -2.f * kLog2e * 0.7978845608028654f));
    }
#pragma unroll
    for (int i = 0; i < N; ++i) top = fmaxf(top, d[i]);
    if (top <= kGateLimit) {
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = gate_quotient(z[i], d[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) z[i] = activate(kind, z[i]);
    }
  } else if (kind == MIE_ACT_RELU) {
#pragma unroll
    for (int i = 0; i < N; ++i) z[i] = activate(MIE_ACT_RELU, z[i]);
  }
}

// Any alignment and size: 64 rows x 64 columns a block, operands by single loads through shared memory, mma.sync.
constexpr int kAnyTile = 64, kAnyK = 32;

template <bool kRouted>
__global__ void __launch_bounds__(128) product_any_kernel(const Product p) {
  __shared__ __align__(16) __nv_bfloat16 sx[kAnyTile][kAnyK + 8];
  __shared__ __align__(16) __nv_bfloat16 sw[2][kAnyTile][kAnyK + 8];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  chain_release();
  chain_wait();
  const int col0 = (int)blockIdx.x * kAnyTile;
  int tile = (int)blockIdx.y;
  const int tiles = kRouted ? *p.tile_count : (p.m + kAnyTile - 1) / kAnyTile;
  const int halves = p.gated ? 2 : 1;
  for (; tile < tiles; tile += gridDim.y) {
    RowTile rows{0, tile * kAnyTile, p.m - tile * kAnyTile < kAnyTile ? p.m - tile * kAnyTile : kAnyTile, 0};
    if (kRouted) rows = p.tiles[tile];
    const __nv_bfloat16* w = p.w + (long long)rows.expert * p.w_expert;
    float acc[2][8][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int i = 0; i < 8; ++i) acc[h][i][0] = acc[h][i][1] = acc[h][i][2] = acc[h][i][3] = 0.f;
    for (int k0 = 0; k0 < p.k; k0 += kAnyK) {
      __syncthreads();
      for (int i = threadIdx.x; i < kAnyTile * kAnyK; i += 128) {
        const int r = i / kAnyK, c = i % kAnyK;
        const bool in = k0 + c < p.k;
        long long row = rows.first + r;
        if (kRouted && r < rows.count && p.source != nullptr) row = p.source[row] / p.source_divisor;
        sx[r][c] = in && r < rows.count ? p.x[row * p.ldx + k0 + c] : __float2bfloat16_rn(0.f);
        for (int h = 0; h < halves; ++h)
          sw[h][r][c] = in && col0 + r < p.n ? w[(long long)(h * p.n + col0 + r) * p.ldw + k0 + c] : __float2bfloat16_rn(0.f);
      }
      __syncthreads();
#pragma unroll
      for (int kk = 0; kk < kAnyK; kk += 16) {
        const uint32_t* a_top = reinterpret_cast<const uint32_t*>(&sx[warp * 16 + g][kk]);
        const uint32_t* a_low = reinterpret_cast<const uint32_t*>(&sx[warp * 16 + g + 8][kk]);
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          if (h >= halves) break;
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const uint32_t* b = reinterpret_cast<const uint32_t*>(&sw[h][i * 8 + g][kk]);
            Mma16816<__nv_bfloat16>::run(acc[h][i], a_top[t], a_low[t], a_top[t + 4], a_low[t + 4], b[t], b[t + 4]);
          }
        }
      }
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int r = warp * 16 + g + 8 * (j >> 1), col = col0 + i * 8 + 2 * t + (j & 1);
        if (r >= rows.count || col >= p.n) continue;
        float v = acc[0][i][j], u = acc[1][i][j];
        if (p.bias != nullptr) {
          v += __bfloat162float(p.bias[col]);
          if (p.gated) u += __bfloat162float(p.bias[p.n + col]);
        }
        v = activate(p.activation, v);
        if (p.gated) v *= u;
        const long long sorted = rows.first + r;
        if (kRouted && p.factor != nullptr) v *= p.factor[p.source[sorted]];
        if (p.residual != nullptr) v += __bfloat162float(p.residual[sorted * p.ldr + col]);
        if (p.wide)
          reinterpret_cast<float*>(p.y)[sorted * p.ldy + col] = v;
        else
          reinterpret_cast<__nv_bfloat16*>(p.y)[sorted * p.ldy + col] = __float2bfloat16_rn(v);
      }
    }
  }
}

}  // namespace
}  // namespace mie
