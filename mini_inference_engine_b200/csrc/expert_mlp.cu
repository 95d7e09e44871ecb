// The gated feed-forward of routed experts:
//
//   y[t] = res[t] + sum_j w[t, j] D_e (act(G_e x[t]) * (U_e x[t])),   e = ids[t, j]
//
// Up to 32 tokens two launches (product_narrow.cuh).  More of them:
//
//   expert_plan_kernel     sorts the (token, choice) pairs by expert and cuts every expert's rows into tiles
//   gate and up product    rows of x gathered by pair; activation, gate and the pair's weight in the epilogue; one rounding to
//                          bf16, which the tensor cores take
//   down product           a row of sums per pair, as fp16 with an exponent per 32 entries: as bf16 the sum over the pairs would
//                          lose as much again as by the hidden rows' rounding, as fp32 its rows would be twice the bytes
//   expert_combine_kernel  adds a token's rows and the residual
//
// 8192 tokens of 2048 x 768, 8 of 128 experts (us, one after the other without a launch chain): 14, 304 to 328, 196 to 207, 86.
// The products are bound as product_wide.cuh says (the down product also by its 268 MB of rows, which HBM takes beside the weights); the
// sum moves its 340 MB at 0.6 of the copy rate.  Together 620 us in a burst, 715 to 780 back to back; the products' floor is 380.
//
// A pair's order among its expert's rows is whatever the counters gave; every row of a product is computed by itself, so
// the results do not depend on it.  Ids outside [0, experts) take no part: -1 says "no expert", others also set a status bit.
#include "product_narrow.cuh"
#include "product_wide.cuh"
#include "products.cuh"
#include "rows.cuh"

namespace mie {
namespace {

struct PlanParams {
  IndexView ids;  // [tokens, top_k]
  int pairs, top_k, experts, tile_rows;
  int* order;     // [pairs] sorted row -> pair
  int* position;  // [pairs] pair -> sorted row, -1 for a pair that takes no part
  RowTile* tiles;
  int* tile_count;
  int* status;
  int dense_ids;  // int32 without gaps, 16-byte aligned
};

constexpr int kPlanThreads = 1024;

__device__ __forceinline__ uint32_t cluster_rank() {
  uint32_t r;
  asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
  return r;
}
__device__ __forceinline__ void plan_cluster_sync() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ int ld_cluster_int(const int* local, uint32_t rank) {
  uint32_t remote;
  int v;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  asm volatile("ld.shared::cluster.s32 %0, [%1];" : "=r"(v) : "r"(remote) : "memory");
  return v;
}

// Sum of `v` over the threads before this one; one value per thread, at most 1024 threads.
__device__ __forceinline__ int block_scan_before(int v, int* warp_sums) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  int sum = v;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int other = __shfl_up_sync(0xffffffffu, sum, o);
    if (lane >= o) sum += other;
  }
  if (lane == 31) warp_sums[warp] = sum;
  __syncthreads();
  if (warp == 0) {
    int s = lane < (int)(blockDim.x >> 5) ? warp_sums[lane] : 0;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, s, o);
      if (lane >= o) s += other;
    }
    warp_sums[lane] = s;
  }
  __syncthreads();
  const int before = (warp > 0 ? warp_sums[warp - 1] : 0) + sum - v;
  __syncthreads();  // warp_sums may be used again
  return before;
}

// Four consecutive pairs' experts, -1 for none.
__device__ __forceinline__ void plan_ids(const PlanParams& p, int i, int end, int (&e)[4]) {
  if (p.dense_ids && i + 4 <= end) {
    const int4 v = *reinterpret_cast<const int4*>(reinterpret_cast<const int*>(p.ids.ptr) + i);
    e[0] = v.x, e[1] = v.y, e[2] = v.z, e[3] = v.w;
  } else {
    int row = i / p.top_k, j = i - row * p.top_k;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      long long id = -1;
      if (i + u < end) id = p.ids.at(row, j);
      e[u] = id >= 0 && id < p.experts ? (int)id : id == -1 ? -1 : -2;
      if (++j == p.top_k) {
        j = 0;
        ++row;
      }
    }
  }
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    if (e[u] >= p.experts || e[u] < -1) {
      raise_status(p.status, MIE_STATUS_BAD_EXPERT);
      e[u] = -1;
    }
  }
}

// One cluster, or one CTA.  Every CTA counts its part of the pairs by expert in shared memory; a thread per expert adds the
// parts up, and with the offsets from a scan over the experts the pairs get their places.  A pair's place among its expert's in
// the CTA's part is kept in `position` meanwhile.
__global__ void __launch_bounds__(kPlanThreads) expert_plan_kernel(const PlanParams p) {
  __shared__ int count[MIE_MAX_EXPERTS], place[MIE_MAX_EXPERTS], warp_sums[32];
  const uint32_t rank = cluster_rank(), ranks = gridDim.x;
  const int fours = (p.pairs + 3) / 4;
  const int begin = (int)((long long)fours * rank / ranks) * 4, stop = (int)((long long)fours * (rank + 1) / ranks) * 4;
  const int end = stop < p.pairs ? stop : p.pairs;
  chain_release();
  for (int e = threadIdx.x; e < p.experts; e += kPlanThreads) count[e] = 0;
  __syncthreads();
  chain_wait();
  constexpr int kHeld = 2;  // fours of a thread whose experts and places stay in registers: pairs up to 8192 a CTA
  int held_e[kHeld][4], held_at[kHeld][4];
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = begin + ((int)threadIdx.x + h * kPlanThreads) * 4;
#pragma unroll
    for (int u = 0; u < 4; ++u) held_e[h][u] = -1;
    if (i < end) plan_ids(p, i, end, held_e[h]);
  }
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
#pragma unroll
    for (int u = 0; u < 4; ++u) held_at[h][u] = held_e[h][u] >= 0 ? atomicAdd(&count[held_e[h][u]], 1) : -1;
  }
  for (int i = begin + ((int)threadIdx.x + kHeld * kPlanThreads) * 4; i < end; i += kPlanThreads * 4) {
    int e[4];
    plan_ids(p, i, end, e);
#pragma unroll
    for (int u = 0; u < 4; ++u)
      if (i + u < end) p.position[i + u] = e[u] >= 0 ? atomicAdd(&count[e[u]], 1) : -1;
  }
  if (ranks > 1)
    plan_cluster_sync();
  else
    __syncthreads();
  const int e = threadIdx.x;
  int total = 0, before = 0;
  if (e < p.experts) {
    if (ranks == 1) {
      total = count[e];
    } else {
      for (uint32_t r = 0; r < ranks; ++r) {
        const int c = ld_cluster_int(&count[e], r);
        if (r < rank) before += c;
        total += c;
      }
    }
  }
  const int first = block_scan_before(total, warp_sums);
  if (e < p.experts) place[e] = first + before;
  if (rank == 0) {
    // As few tiles as hold the expert's rows, about equally long, in multiples of 16.
    int tiles = (total + p.tile_rows - 1) / p.tile_rows;
    const int rows = tiles > 0 ? ((total + tiles - 1) / tiles + 15) / 16 * 16 : 16;
    tiles = (total + rows - 1) / rows;
    const int tile = block_scan_before(tiles, warp_sums);
    for (int i = 0; i < tiles; ++i) {
      const int left = total - i * rows;
      p.tiles[tile + i] = RowTile{e, first + i * rows, left < rows ? left : rows, 0};
    }
    if (e == kPlanThreads - 1) *p.tile_count = tile + tiles;
  }
  __syncthreads();
#pragma unroll
  for (int h = 0; h < kHeld; ++h) {
    const int i = begin + ((int)threadIdx.x + h * kPlanThreads) * 4;
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u >= end) continue;
      const int sorted = held_at[h][u] >= 0 ? place[held_e[h][u]] + held_at[h][u] : -1;
      if (sorted >= 0) p.order[sorted] = i + u;
      held_at[h][u] = sorted;
    }
    if (i + 4 <= end) {
      *reinterpret_cast<int4*>(p.position + i) = make_int4(held_at[h][0], held_at[h][1], held_at[h][2], held_at[h][3]);
    } else {
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (i + u < end) p.position[i + u] = held_at[h][u];
    }
  }
  for (int i = begin + ((int)threadIdx.x + kHeld * kPlanThreads) * 4; i < end; i += kPlanThreads * 4) {
    int expert[4];
    plan_ids(p, i, end, expert);
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      if (i + u >= end || expert[u] < 0) continue;
      const int sorted = place[expert[u]] + p.position[i + u];
      p.order[sorted] = i + u;
      p.position[i + u] = sorted;
    }
  }
  if (ranks > 1) plan_cluster_sync();  // no CTA leaves while another may still read its counts
}

struct CombineParams {
  const void* rows;          // [pairs, width] in sorted order: fp32, or fp16 with
  const int8_t* exponents;   // [pairs, exponent_ld], one per 32 entries: value = entry / 2^exponent
  int exponent_ld;
  const int* position;       // [tokens, top_k] sorted row of a pair or -1
  const __nv_bfloat16* residual;
  long long ldr;
  __nv_bfloat16* y;
  long long ldy;
  int tokens, top_k, width;
};

// The residual and the pairs' rows, added in the order of the choices.
__global__ void __launch_bounds__(256) expert_combine_any_kernel(const CombineParams p) {
  chain_release();
  chain_wait();
  const long long total = (long long)p.tokens * p.width;
  for (long long i = (long long)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (long long)gridDim.x * blockDim.x) {
    const long long t = i / p.width;
    const int c = (int)(i - t * p.width);
    float sum = p.residual != nullptr ? __bfloat162float(p.residual[t * p.ldr + c]) : 0.f;
    for (int j = 0; j < p.top_k; ++j) {
      const long long row = p.position[t * p.top_k + j];
      if (row >= 0) sum += reinterpret_cast<const float*>(p.rows)[row * p.width + c];
    }
    p.y[t * p.ldy + c] = __float2bfloat16_rn(sum);
  }
}

// Eight entries a thread, eight pairs' rows in flight, the next token's positions read ahead; bound by HBM.
__global__ void __launch_bounds__(256) expert_combine_kernel(const CombineParams p) {
  chain_release();
  const bool vec_y = p.ldy % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
  const bool vec_r = p.ldr % 8 == 0 && (reinterpret_cast<uintptr_t>(p.residual) & 15) == 0;
  const int lane = threadIdx.x & 31, step = gridDim.x * blockDim.y;
  chain_wait();
  int t = blockIdx.x * blockDim.y + threadIdx.y;
  // Lane j of a warp: the j-th position of its token (blockDim.x is a multiple of 32).
  int next = t < p.tokens && lane < p.top_k ? p.position[(long long)t * p.top_k + lane] : -1;
  for (; t < p.tokens; t += step) {
    const int position = next;
    if (t + step < p.tokens) next = lane < p.top_k ? p.position[(long long)(t + step) * p.top_k + lane] : -1;
    for (int c0 = 0; c0 < p.width; c0 += blockDim.x * 8) {
      const int c = c0 + threadIdx.x * 8;
      const bool in = c < p.width;
      uint4 residual = make_uint4(0, 0, 0, 0);
      float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
      if (p.residual != nullptr && in) {
        const __nv_bfloat16* r = p.residual + (long long)t * p.ldr + c;
        if (vec_r) {
          residual = __ldcs(reinterpret_cast<const uint4*>(r));
        } else {
#pragma unroll
          for (int n = 0; n < 8; ++n) sum[n] = __bfloat162float(r[n]);
        }
      }
      for (int j0 = 0; j0 < p.top_k; j0 += 8) {
        uint4 raw[8];
        int exponent[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const int row = j0 + u < 32 ? __shfl_sync(0xffffffffu, position, (j0 + u) & 31) : -1;
          raw[u] = make_uint4(0, 0, 0, 0);
          exponent[u] = 0;
          if (row >= 0 && in) {
            raw[u] = __ldcs(reinterpret_cast<const uint4*>(reinterpret_cast<const __half*>(p.rows) + (long long)row * p.width + c));
            exponent[u] = p.exponents[(long long)row * p.exponent_ld + c / 32];
          }
        }
        if (j0 == 0 && p.residual != nullptr && vec_r) {
          const uint32_t w[4] = {residual.x, residual.y, residual.z, residual.w};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 f = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&w[n]));
            sum[2 * n] = f.x;
            sum[2 * n + 1] = f.y;
          }
        }
#pragma unroll
        for (int u = 0; u < 8; ++u) {
          const float scale = __uint_as_float((uint32_t)(127 - exponent[u]) << 23);
          const uint32_t w[4] = {raw[u].x, raw[u].y, raw[u].z, raw[u].w};
#pragma unroll
          for (int n = 0; n < 4; ++n) {
            const float2 f = __half22float2(*reinterpret_cast<const __half2*>(&w[n]));
            sum[2 * n] = fmaf(f.x, scale, sum[2 * n]);
            sum[2 * n + 1] = fmaf(f.y, scale, sum[2 * n + 1]);
          }
        }
      }
      if (!in) continue;
      __nv_bfloat16* y = p.y + (long long)t * p.ldy + c;
      if (vec_y) {
        Vec<__nv_bfloat16, 8>::store(y, sum);
      } else {
#pragma unroll
        for (int n = 0; n < 8; ++n) y[n] = __float2bfloat16_rn(sum[n]);
      }
    }
  }
}

constexpr int kMostParts = 320;  // CTAs of a few rows' down product that leave a part of the sums

// Where the parts of the scratch begin.
struct Scratch {
  long long order, position, tiles, tile_count, hidden, exponents, rows, total;
  Scratch(long long tokens, int top_k, int experts, int width, int ff) {
    const long long pairs = tokens * top_k;
    total = 0;
    order = take((pairs > (width + 127) / 128 ? pairs : (width + 127) / 128) * 4);
    position = take(pairs * 4);
    tiles = take(most_tiles(pairs, experts, kAnyTile) * (long long)sizeof(RowTile));
    tile_count = take(4);
    // Few rows: a hidden row of every token for every expert in use.
    const long long few = tokens > kFewRoutedRows ? 0 : (pairs < experts ? pairs : experts) * (tokens > 16 ? 32 : 16);
    hidden = take((pairs > few ? pairs : few) * ff * 2);
    exponents = take(pairs * exponent_ld(width));
    // Few rows: the parts of the down product, at most one CTA's an SM or one of every tile.
    const long long tiles = (width + 127) / 128, ctas = tiles > kMostParts ? tiles : kMostParts;
    const long long parts = tokens > kFewRoutedRows ? 0 : ctas * (tokens > 16 ? 32 : 16) * 128 * 4;
    rows = take(pairs * width * 4 > parts ? pairs * width * 4 : parts);
  }
  long long take(long long bytes) {
    const long long at = total;
    total += (bytes + 255) / 256 * 256;
    return at;
  }
  // Every expert's rows in tiles of at least half of tile_rows but one.
  static long long most_tiles(long long pairs, int experts, int tile_rows) {
    return 2 * (pairs / tile_rows) + (pairs < experts ? pairs : experts);
  }
  static int exponent_ld(int width) { return (width + 31) / 32; }
};

int launch_plan(const PlanParams& plan, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3(plan.pairs > 4096 ? 8 : 1);
  config.blockDim = dim3(kPlanThreads);
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = config.gridDim.x;
  attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = chained_launch_enabled() ? 2 : 1;
  MIE_CUDA(cudaLaunchKernelEx(&config, expert_plan_kernel, plan));
  MIE_LAUNCH_CHECK("expert_plan_kernel");
  return MIE_OK;
}

// Parts of a few rows' down product that meet in global memory, 0: it goes by clusters.  16 clusters of eight, a CTA an SM at
// most, do not keep HBM busy, two CTAs an SM do; but the last one to arrive adds 5 us.  The layer in us, clusters and parts,
// width 2048 and 128 experts of 768: 1 token 22.6 and 27.9, 4 59.6 and 60.5, 8 84 and 79, 32 160 and 144; where clusters of eight
// come to two CTAs an SM (width 4096, 8 experts of 2048), 2 tokens 39.9 and 41.9, 32 78.8 and 82.0.
int few_parts(int width, long long pairs, int cluster) {
  const int tiles = (width + 127) / 128, ctas = 2 * sm_count() < kMostParts ? 2 * sm_count() : kMostParts, parts = ctas / tiles;
  if (pairs <= 40 || tiles * cluster >= 1.3 * sm_count() || parts <= cluster) return 0;
  return parts > 24 ? 24 : parts;
}

// Few rows: every expert in use for all of them (see product_narrow.cuh).
template <int BN>
int launch_routed_few(const Product& up, const Product& out, FewParams q, cudaStream_t stream) {
  const int rows = up.m;
  CUtensorMap map_w, map_x;
  q.p = up;
  q.weight_tiles = (up.n + 63) / 64;
  q.down_tiles = (out.n + 127) / 128;
  const long long pairs = (long long)rows * q.top_k, most = pairs < q.experts ? pairs : q.experts;
  if (int rc = few_weight_map(&map_w, up, q.experts, 64)) return rc;
  if (int rc = row_map(&map_x, up, rows, BN)) return rc;
  const long long tiles = most * q.weight_tiles, slots = 2ll * sm_count();
  const int split = few_split(tiles, (up.k + 63) / 64, 2);
  if (int rc = launch_few<BN, Few::kUp, true>(map_w, map_x, q, split == 1 && tiles > slots ? slots : tiles, split, 1, stream))
    return rc;
  q.p = out;
  q.weight_tiles = q.down_tiles;
  if (int rc = few_weight_map(&map_w, out, q.experts, 128)) return rc;
  const uint64_t dims[3] = {(uint64_t)out.k, (uint64_t)BN, (uint64_t)most};
  const uint64_t strides[2] = {(uint64_t)out.ldx * 2, (uint64_t)out.ldx * 2 * BN};
  const uint32_t box[3] = {64, (uint32_t)BN, 1};
  if (int rc = operand_map_bf16(&map_x, 3, out.x, dims, strides, box)) return rc;
  const int cluster = few_split(q.weight_tiles, (int)most * ((out.k + 63) / 64), 2), parts = few_parts(out.n, pairs, cluster);
  if (parts == 0) q.parts = nullptr;
  return launch_few<BN, Few::kDown, false>(map_w, map_x, q, q.weight_tiles, parts > 0 ? parts : cluster, 1, stream);
}

int launch_any(const Product& p, long long tiles, cudaStream_t stream) {
  MIE_CUDA(launch_chained(product_any_kernel<true>,
                          dim3((unsigned)((p.n + kAnyTile - 1) / kAnyTile), (unsigned)(tiles < 65535 ? tiles : 65535)),
                          dim3(128), 0, stream, p));
  MIE_LAUNCH_CHECK("product_any_kernel");
  return MIE_OK;
}

}  // namespace
}  // namespace mie

using namespace mie;

extern "C" int64_t mie_expert_scratch_bytes(int32_t tokens, int32_t top_k, int32_t experts, int32_t width, int32_t ff) {
  if (tokens < 0 || top_k < 1 || experts < 1 || width < 1 || ff < 1 || width > MIE_MAX_PRODUCT || ff > 1 << 30) return 0;
  return Scratch(tokens, top_k, experts, width, ff).total;
}

extern "C" int mie_expert_mlp(const void* x, int64_t ldx, mie_index_t ids, const float* weights, const void* gate_up,
                              int64_t gate_up_row, int64_t gate_up_expert, const void* down, int64_t down_row,
                              int64_t down_expert, const void* residual, int64_t ldr, void* y, int64_t ldy,
                              int32_t tokens, int32_t top_k, int32_t experts, int32_t width, int32_t ff,
                              int32_t activation, void* scratch, int64_t scratch_bytes, int32_t* status, void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  MIE_CHECK_ARG(x && ids.ptr && weights && gate_up && down && y && scratch, "null pointer");
  MIE_CHECK_ARG(tokens >= 0 && width >= 1 && width <= MIE_MAX_PRODUCT && ff >= 1 && ff <= 1 << 30 && experts >= 1 &&
                    experts <= MIE_MAX_EXPERTS && top_k >= 1 && top_k <= MIE_MAX_TOP_K,
                "invalid sizes: %d tokens of %d, %d of %d experts of %d", tokens, width, top_k, experts, ff);
  MIE_CHECK_ARG((long long)tokens * top_k < (1ll << 30), "too many (token, expert) pairs");
  MIE_CHECK_ARG(ldx >= width && gate_up_row >= width && down_row >= ff && ldy >= width && (!residual || ldr >= width),
                "a row is longer than its stride");
  MIE_CHECK_ARG(activation >= MIE_ACT_NONE && activation <= MIE_ACT_RELU, "unknown activation %d", activation);
  const int pairs = tokens * top_k;
  if (tokens == 0) return MIE_OK;
  const Scratch s(tokens, top_k, experts, width, ff);
  MIE_CHECK_ARG(scratch_bytes >= s.total, "scratch of %lld bytes, %lld needed", (long long)scratch_bytes, s.total);
  MIE_CHECK_ARG((reinterpret_cast<uintptr_t>(scratch) & 255) == 0, "scratch must be 256-byte aligned");
  uint8_t* base = (uint8_t*)scratch;
  int* order = (int*)(base + s.order);

  Product up = {};
  up.x = (const __nv_bfloat16*)x, up.ldx = ldx;
  up.w = (const __nv_bfloat16*)gate_up, up.ldw = gate_up_row, up.w_expert = gate_up_expert;
  up.y = base + s.hidden, up.ldy = ff;
  up.m = pairs, up.n = ff, up.k = width;
  up.activation = activation, up.gated = 1, up.status = status;
  up.tiles = (RowTile*)(base + s.tiles), up.tile_count = (int*)(base + s.tile_count);
  up.source = order, up.source_divisor = top_k, up.factor = weights;

  Product out = {};
  out.x = (const __nv_bfloat16*)(base + s.hidden), out.ldx = ff;
  out.w = (const __nv_bfloat16*)down, out.ldw = down_row, out.w_expert = down_expert;
  out.y = base + s.rows, out.ldy = width;
  out.m = pairs, out.n = width, out.k = ff;
  out.status = status;
  out.tiles = up.tiles, out.tile_count = up.tile_count;

  CombineParams combine{base + s.rows, (const int8_t*)(base + s.exponents), s.exponent_ld(width), (const int*)(base + s.position),
                        (const __nv_bfloat16*)residual, ldr, (__nv_bfloat16*)y, ldy, tokens, top_k, width};

  const bool wide = wide_takes(up) && wide_takes(out) && direct_takes(out);
  if (wide && tokens <= kFewRoutedRows) {
    FewParams few = {};
    few.parts = (float*)(base + s.rows), few.arrived = order;
    few.ids = IndexView(ids), few.weights = weights, few.top_k = top_k, few.experts = experts;
    up.m = out.m = tokens;
    out.y = y, out.ldy = ldy, out.residual = (const __nv_bfloat16*)residual, out.ldr = ldr;
    return tokens <= 16 ? launch_routed_few<16>(up, out, few, stream) : launch_routed_few<32>(up, out, few, stream);
  }
  const int tile_rows = wide ? kWideRows : kAnyTile;
  const long long tiles = s.most_tiles(pairs, experts, tile_rows);
  const PlanParams plan{IndexView(ids), pairs, top_k, experts, tile_rows, order, (int*)(base + s.position),
                        (RowTile*)(base + s.tiles), (int*)(base + s.tile_count), status,
                        !ids.is64 && ids.stride1 == 1 && ids.stride0 == top_k && (reinterpret_cast<uintptr_t>(ids.ptr) & 15) == 0};
  if (int rc = launch_plan(plan, stream)) return rc;
  if (!wide) {
    out.wide = 1;
    if (int rc = launch_any(up, tiles, stream)) return rc;
    if (int rc = launch_any(out, tiles, stream)) return rc;
    const long long blocks = ((long long)tokens * width + 255) / 256, most = 16ll * sm_count();
    MIE_CUDA(launch_chained(expert_combine_any_kernel, dim3((unsigned)(blocks < most ? blocks : most)), dim3(256), 0, stream,
                            combine));
    MIE_LAUNCH_CHECK("expert_combine_any_kernel");
    return MIE_OK;
  }
  WideParams q = {};
  WeightMaps maps;
  CUtensorMap map_x;
  q.p = up;
  q.weight_tiles = (ff + 127) / 128;
  if (int rc = weight_maps(&maps, up, experts, false)) return rc;
  if (int rc = row_map(&map_x, up, tokens, 1)) return rc;
  if (int rc = launch_wide<Rows::kUp, true, false>(maps, map_x, q, tiles * q.weight_tiles, 1, stream)) return rc;
  q.p = out;
  q.weight_tiles = (width + 255) / 256;
  q.x_box = 32;
  q.exponents = (int8_t*)(base + s.exponents);
  q.exponent_ld = s.exponent_ld(width);
  if (int rc = weight_maps(&maps, out, experts, true)) return rc;
  if (int rc = row_map(&map_x, out, pairs, q.x_box)) return rc;
  if (int rc = launch_wide<Rows::kDown, false, true>(maps, map_x, q, tiles * q.weight_tiles, 1, stream)) return rc;
  const int lanes = width / 8 < 256 ? (width / 8 + 31) / 32 * 32 : 256, rows_per_block = 256 / lanes;
  const long long blocks = ((long long)tokens + rows_per_block - 1) / rows_per_block, most = 16ll * sm_count();
  MIE_CUDA(launch_chained(expert_combine_kernel, dim3((unsigned)(blocks < most ? blocks : most)),
                          dim3((unsigned)lanes, (unsigned)rows_per_block), 0, stream, combine));
  MIE_LAUNCH_CHECK("expert_combine_kernel");
  return MIE_OK;
}
