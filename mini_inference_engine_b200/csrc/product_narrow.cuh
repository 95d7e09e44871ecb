// Products of few rows: the weights are streamed once, 128 rows of them a CTA as the M of a tcgen05 accumulator whose N are the
// BN rows of x.  Bound by HBM, and by the time from the kernel before to the first weights and from the last weights to the
// end.  Where the weight has too few tiles to fill the GPU, K is cut in parts: across a cluster of up to 8 CTAs, whose sums meet
// in shared memory, or (kDown) over two CTAs an SM, whose sums meet in global memory, added by the last one to come; in either
// case in the order of the parts.
//
//   kDense  y = act(x W^T + b) + res, gated or not
//   kUp     routed: every expert that any row is sent to, for all rows: hidden[u][row] = act(G x) * (U x), u the expert's
//           place among those in use.  Rows of x that are not sent there are computed too (the weights are what counts), not
//           used.
//   kDown   routed: y[row] = res + sum_u w[row, u] D_u hidden[u][row].  The sum over the experts is one long K, cut in parts (see
//           few_parts); where an expert ends its part is taken out of tensor memory and added, with its weights, to the rows
//           that are sent there and to no others (an expert's infinities stay with its rows).
//
// Measured: 1 row of 12288 x 2048 gated 12.0 us, 24 rows of 2560 x 9728 12.8 (their bytes 7.7 each): about 2 us from the start to
// the first weights, 1.5 to 3 from the last ones to the end, growing with the rows, and what two CTAs an SM with 100 KB of ring
// each get from HBM between.  A routed layer of 128 experts (2048 x 768, 8 a token) 22.4 us for 1 token (11.6), 79 for 8 (65 if
// their experts are spread evenly, fewer are read where some are favoured), 146 for 32 (121 by the same count).
//
// Which experts are in use every CTA finds out by itself from the ids, a few hundred at most.  kUp lets the kernel after it
// start behind its own wait for the kernels before: kDown may read the ids, and ask for its first weights, while kUp runs.
#pragma once

#include "products.cuh"
#include "umma.cuh"

namespace mie {
namespace {

enum class Few { kDense, kUp, kDown };

constexpr int kFewThreads = 192;     // 4 finishing warps, TMA producer, MMA issuer
constexpr int kFewRoutedRows = 32;   // most rows of the routed form
constexpr int kFewPairs = kFewRoutedRows * MIE_MAX_TOP_K;

template <int BN, Few kKind>
struct FewSmem {
  static constexpr int kStageBytes = 128 * 128 + BN * 128;
  static constexpr int kCtasPerSm = 2;  // one CTA's ring alone does not cover HBM's latency
  static constexpr int kParkBytes = BN * 128 * 4;  // kUp: its own, the others' is the idle ring
  static constexpr int kRouting = kKind == Few::kDense ? 0 : kFewPairs * 6 + MIE_MAX_EXPERTS * 2 + 256;
  static constexpr int kExtra = kRouting + (kKind == Few::kUp ? kParkBytes : 0);
  static constexpr int kStages = (111 * 1024 - kExtra) / kStageBytes;
  static constexpr int kAcc = kKind == Few::kDown ? 4 : kKind == Few::kUp ? 2 : 1;  // accumulators in tensor memory
  static constexpr int kAccColumns = BN < 32 ? 32 : BN;
  static constexpr int kTotal = kStages * kStageBytes + kExtra + (2 * kStages + 2 * kAcc) * 8 + 16 + 1024;
  static_assert(kTotal <= 113 * 1024, "shared memory of an SM");
  static_assert(kStages * kStageBytes >= kParkBytes, "the ring also parks the fp32 sums");
};

struct FewParams {
  Product p;
  // Routed.
  IndexView ids;  // [rows, top_k]
  const float* weights;
  int top_k, experts, weight_tiles;
  float* parts;    // kDown: [tiles][split][BN][128], null: the parts are a cluster
  int* arrived;    // kDown: [tiles], zeroed by kUp
  int down_tiles;  // kUp: how many those are
};

// The experts in use, in the same order for kUp and kDown, and the pairs' experts and weights, in shared memory.
struct Routing {
  int16_t* used;      // [MIE_MAX_EXPERTS]
  int16_t* expert;    // [rows * top_k], -1: none
  float* weight;      // [rows * top_k]
  uint32_t* bitmap;   // [32]
  int* count;
};
__device__ __forceinline__ Routing routing_at(uint8_t* base) {
  Routing r;
  r.weight = reinterpret_cast<float*>(base);
  r.used = reinterpret_cast<int16_t*>(base + kFewPairs * 4);
  r.expert = r.used + MIE_MAX_EXPERTS;
  r.bitmap = reinterpret_cast<uint32_t*>(r.expert + kFewPairs);
  r.count = reinterpret_cast<int*>(r.bitmap + 32);
  return r;
}
__device__ __forceinline__ int find_routing(const Routing& r, const FewParams& q, bool report) {
  const int pairs = q.p.m * q.top_k, tid = threadIdx.x;
  if (pairs <= 32) {  // one warp, in the order of the pairs
    if (tid < 32) {
      const int row = tid / q.top_k;
      const long long e = tid < pairs ? q.ids.at(row, tid - row * q.top_k) : -1;
      const bool valid = e >= 0 && e < q.experts;
      if (!valid && e != -1 && report) raise_status(q.p.status, MIE_STATUS_BAD_EXPERT);
      const int expert = valid ? (int)e : -1;
      const uint32_t same = __match_any_sync(0xffffffffu, expert);
      const bool first = valid && __ffs(same) - 1 == tid;
      const uint32_t firsts = __ballot_sync(0xffffffffu, first);
      if (first) r.used[__popc(firsts & ((1u << tid) - 1u))] = (int16_t)expert;
      if (tid < pairs) {
        r.expert[tid] = (int16_t)expert;
        r.weight[tid] = q.weights[tid];
      }
      if (tid == 0) *r.count = __popc(firsts);
    }
    __syncthreads();
    return *r.count;
  }
  if (tid < 32) r.bitmap[tid] = 0;
  __syncthreads();
  for (int i = tid; i < pairs; i += kFewThreads) {
    const int row = i / q.top_k;
    const long long e = q.ids.at(row, i - row * q.top_k);
    const bool valid = e >= 0 && e < q.experts;
    if (!valid && e != -1 && report) raise_status(q.p.status, MIE_STATUS_BAD_EXPERT);
    r.expert[i] = valid ? (int16_t)e : (int16_t)-1;
    r.weight[i] = q.weights[i];
    if (valid) atomicOr(&r.bitmap[e >> 5], 1u << (e & 31));
  }
  __syncthreads();
  if (tid < 32) {
    uint32_t word = r.bitmap[tid];
    int before = __popc(word);
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int other = __shfl_up_sync(0xffffffffu, before, o);
      if (tid >= o) before += other;
    }
    if (tid == 31) *r.count = before;
    before -= __popc(word);
    for (; word != 0; word &= word - 1) r.used[before++] = (int16_t)(tid * 32 + __ffs(word) - 1);
  }
  __syncthreads();
  return *r.count;
}

// Four channels of a row from the parked sums of all CTAs, in rank order.
template <int kSplit>
__device__ __forceinline__ float4 sum_parts(uint32_t park, int at) {
  float4 part[kSplit];
#pragma unroll
  for (int peer = 0; peer < kSplit; ++peer) {
    if (kSplit == 1)
      asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];"
                   : "=f"(part[0].x), "=f"(part[0].y), "=f"(part[0].z), "=f"(part[0].w)
                   : "r"(park + (uint32_t)at * 4u)
                   : "memory");
    else
      part[peer] = ld_cluster_f4(park + (uint32_t)at * 4u, (uint32_t)peer);
  }
  float4 sum = part[0];
#pragma unroll
  for (int peer = 1; peer < kSplit; ++peer) {
    sum.x += part[peer].x;
    sum.y += part[peer].y;
    sum.z += part[peer].z;
    sum.w += part[peer].w;
  }
  return sum;
}

// The rows of a tile, finished in units of four channels of a row over all threads of the cluster, several units at a time
// (one by one the latencies of the sums, the residual and the activation took 5 us of 128 rows).
template <int BN, Few kKind, bool kGated, int kSplit>
__device__ __forceinline__ void finish_rows(const FewParams& q, uint32_t park, int rank, int rows, long long to0, int channel0) {
  constexpr int kFours = kGated ? 16 : 32;
  constexpr int kBatch = BN == 16 || kSplit == 8 ? 1 : kSplit == 4 ? 2 : 4;
  const Product& p = q.p;
  const bool has_residual = kKind != Few::kUp && p.residual != nullptr;
  const bool vec_residual = has_residual && p.ldr % 4 == 0 && (reinterpret_cast<uintptr_t>(p.residual) & 7) == 0;
  const bool vec_y = p.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0;
  const int four = (int)threadIdx.x % kFours, channel = channel0 + four * 4;  // the same for all of a thread's units
  const int valid = p.n - channel < 4 ? p.n - channel : 4;
  if (valid <= 0) return;
  float bias[4] = {0.f, 0.f, 0.f, 0.f}, bias_up[4] = {0.f, 0.f, 0.f, 0.f};
  if (kKind == Few::kDense && p.bias != nullptr) {
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      if (j >= valid) break;
      bias[j] = __bfloat162float(p.bias[channel + j]);
      if (kGated) bias_up[j] = __bfloat162float(p.bias[p.n + channel + j]);
    }
  }
  constexpr int kStep = 128 / kFours * kSplit;  // rows that the cluster finishes at a time
  for (int first = rank * (128 / kFours) + (int)threadIdx.x / kFours; first < rows; first += kBatch * kStep) {
    float v[4 * kBatch], u[kBatch][4], r[kBatch][4];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      const int row = first + b * kStep < rows ? first + b * kStep : first;
      const float4 s = sum_parts<kSplit>(park, row * 128 + four * 4);
      v[4 * b] = s.x + bias[0], v[4 * b + 1] = s.y + bias[1], v[4 * b + 2] = s.z + bias[2], v[4 * b + 3] = s.w + bias[3];
      if (kGated) {
        const float4 up = sum_parts<kSplit>(park, row * 128 + 64 + four * 4);
        u[b][0] = up.x + bias_up[0], u[b][1] = up.y + bias_up[1], u[b][2] = up.z + bias_up[2], u[b][3] = up.w + bias_up[3];
      }
#pragma unroll
      for (int j = 0; j < 4; ++j) r[b][j] = 0.f;
      if (has_residual) {
        const __nv_bfloat16* src = p.residual + (to0 + row) * p.ldr + channel;
        if (vec_residual && valid == 4) {
          const uint2 raw = *reinterpret_cast<const uint2*>(src);
          const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.x));
          const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&raw.y));
          r[b][0] = lo.x, r[b][1] = lo.y, r[b][2] = hi.x, r[b][3] = hi.y;
        } else {
#pragma unroll
          for (int j = 0; j < 4; ++j)
            if (j < valid) r[b][j] = __bfloat162float(src[j]);
        }
      }
    }
    if (kKind != Few::kDown) activate_all(p.activation, v);
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
      if (first + b * kStep >= rows) break;
      float o[4];
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = (kGated ? v[4 * b + j] * u[b][j] : v[4 * b + j]) + r[b][j];
      __nv_bfloat16* y = reinterpret_cast<__nv_bfloat16*>(p.y) + (to0 + first + b * kStep) * p.ldy + channel;
      if (vec_y && valid == 4) {
        *reinterpret_cast<uint2*>(y) =
            make_uint2(Mma16816<__nv_bfloat16>::pack(o[0], o[1]), Mma16816<__nv_bfloat16>::pack(o[2], o[3]));
      } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
          if (j < valid) y[j] = __float2bfloat16_rn(o[j]);
      }
    }
  }
}

// grid = (tiles, split, tiles of rows), cluster = (1, split) unless the parts meet in global memory.  Without a split, kUp has as
// many CTAs as run at once, which go through the tiles of all experts without a pause.
template <int BN, Few kKind, bool kGated>
__global__ void __launch_bounds__(kFewThreads, FewSmem<BN, kKind>::kCtasPerSm)
    product_few_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_x, const FewParams q) {
  using S = FewSmem<BN, kKind>;
  constexpr int kStages = S::kStages, kAcc = S::kAcc;
  constexpr int kTmemColumns = kAcc * S::kAccColumns;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* park_at = kKind == Few::kUp ? ring + kStages * S::kStageBytes : ring;
  uint64_t* full_bar =
      reinterpret_cast<uint64_t*>(ring + kStages * S::kStageBytes + (kKind == Few::kUp ? S::kParkBytes : 0));
  uint64_t* empty_bar = full_bar + kStages;
  uint64_t* acc_full = empty_bar + kStages;
  uint64_t* acc_empty = acc_full + kAcc;
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + kAcc);
  const Routing routing = routing_at(reinterpret_cast<uint8_t*>(tmem_slot + 4));
  const Product& p = q.p;
  const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
  const int split = gridDim.y, rank = blockIdx.y;
  const int blocks = (p.k + 63) / 64;  // of an expert's K

  if (warp == 4 && lane == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < kAcc; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 4);
    }
    mbar_fence_init();
    tma_prefetch_desc(&map_w);
    tma_prefetch_desc(&map_x);
  }
  if (warp == 5) {
    tmem_alloc(tmem_slot, kTmemColumns);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  // kDown reads the ids and weights ahead of its wait: kUp, whose hidden rows it waits for, has waited for what wrote them.
  if (kKind != Few::kUp) chain_release();
  if (kKind != Few::kDown) chain_wait();
  if (kKind == Few::kUp) {
    chain_release();
    for (int i = (int)(blockIdx.x * kFewThreads + threadIdx.x); i < q.down_tiles; i += (int)gridDim.x * kFewThreads)
      q.arrived[i] = 0;
  }
  const int used = kKind == Few::kDense ? 1 : find_routing(routing, q, kKind == Few::kUp);

  const int row0 = kKind == Few::kDense ? (int)blockIdx.z * BN : 0, rows = p.m - row0 < BN ? p.m - row0 : BN;
  // The CTA's work: units of `blocks` blocks of K, each with an accumulator of its own.  kUp: tiles blockIdx.x, + gridDim.x, ...
  // of all experts' in use; kDown: the experts in use.
  int units = 1;
  if (kKind == Few::kUp) {
    const int left = used * q.weight_tiles - (int)blockIdx.x;
    units = left <= 0 ? 0 : (left + (int)gridDim.x - 1) / (int)gridDim.x;
  }
  if (kKind == Few::kDown) units = used;
  const int total = units * blocks;
  const int first = (int)((long long)total * rank / split);
  const int count = (int)((long long)total * (rank + 1) / split) - first;
  auto tile_of = [&](int unit) {
    return kKind == Few::kUp ? ((int)blockIdx.x + unit * (int)gridDim.x) % q.weight_tiles : (int)blockIdx.x;
  };
  auto place_of = [&](int unit) {
    return kKind == Few::kUp ? ((int)blockIdx.x + unit * (int)gridDim.x) / q.weight_tiles : kKind == Few::kDown ? unit : 0;
  };

  bool ok = true;
  const uint32_t park = smem_u32(park_at);
  if (warp == 4) {
    if (lane == 0) {
      const uint64_t policy = l2_evict_first_policy();  // weights are streamed once per call
      int requested = 0;
      auto request_weights = [&](int i) {
        const int s = i % kStages, at = first + i;
        const int unit = kKind == Few::kDense ? 0 : at / blocks, b = at - unit * blocks, tile = tile_of(unit);
        const int e = kKind == Few::kDense ? 0 : routing.used[place_of(unit)];
        uint8_t* dst = ring + (size_t)s * S::kStageBytes;
        mbar_expect_tx(&full_bar[s], S::kStageBytes);
        if (kGated) {
          tma_load_3d_hint(dst, &map_w, &full_bar[s], b * 64, tile * 64, e, policy);
          tma_load_3d_hint(dst + 8192, &map_w, &full_bar[s], b * 64, p.n + tile * 64, e, policy);
        } else {
          tma_load_3d_hint(dst, &map_w, &full_bar[s], b * 64, tile * 128, e, policy);
        }
      };
      if (kKind == Few::kDown) {
        for (; requested < count && requested < kStages; ++requested) request_weights(requested);
        chain_wait();
      }
      for (int i = 0; i < count; ++i) {
        const int s = i % kStages, at = first + i;
        if (i >= requested) {
          if (!mbar_wait_bounded(&empty_bar[s], ((i / kStages) & 1u) ^ 1u)) {
            raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
            break;
          }
          request_weights(i);
        }
        uint8_t* dst = ring + (size_t)s * S::kStageBytes + 128 * 128;
        const int unit = kKind == Few::kDense ? 0 : at / blocks, b = at - unit * blocks;
        if (kKind == Few::kDown)
          tma_load_3d(dst, &map_x, &full_bar[s], b * 64, 0, unit);
        else
          tma_load_2d(dst, &map_x, &full_bar[s], b * 64, row0);
      }
    }
    __syncwarp();
  } else if (warp == 5) {
    constexpr uint32_t idesc = instr_desc_bf16(128, BN, 0, 0);
    int part = 0;  // runs of one unit
    for (int i = 0; i < count; ++i) {
      const int s = i % kStages;
      const int in_unit = kKind == Few::kDense ? i : (first + i) % blocks;
      const bool opens = i == 0 || in_unit == 0;
      const bool closes = i == count - 1 || in_unit == blocks - 1;
      const int acc = part % kAcc;
      if (opens && part >= kAcc && !warp_wait_bounded(&acc_empty[acc], ((part / kAcc) & 1u) ^ 1u)) {
        raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
        break;
      }
      if (!warp_wait_bounded(&full_bar[s], (i / kStages) & 1u)) {
        raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
        break;
      }
      tc_fence_after();
      if (elect_one()) {
        const uint32_t a = smem_u32(ring + (size_t)s * S::kStageBytes);
        const uint64_t da = smem_desc_k128(a), db = smem_desc_k128(a + 128 * 128);
#pragma unroll
        for (int k = 0; k < 4; ++k)
          umma_f16(tmem + acc * S::kAccColumns, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc,
                   opens && k == 0 ? 0u : 1u);
        umma_commit(&empty_bar[s]);
        if (closes) umma_commit(&acc_full[acc]);
      }
      __syncwarp();
      if (closes) ++part;
    }
  } else {
    // One weight row a thread.
    const int row = warp * 32 + lane;
    const uint32_t lane_addr = tmem + ((uint32_t)(warp * 32) << 16);
    float sum[BN];
#pragma unroll
    for (int j = 0; j < BN; ++j) sum[j] = 0.f;
    auto take = [&](int part, float (&v)[BN]) {
      const int acc = part % kAcc;
      if (ok && !warp_wait_bounded(&acc_full[acc], (part / kAcc) & 1u)) {
        ok = false;
        raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
      }
      tc_fence_after();
      if constexpr (BN >= 32) {
#pragma unroll
        for (int c = 0; c < BN; c += 32)
          tmem_ld32(lane_addr + acc * S::kAccColumns + c, *reinterpret_cast<float(*)[32]>(&v[c]));
      } else {
        tmem_ld16(lane_addr + acc * S::kAccColumns, *reinterpret_cast<float(*)[16]>(&v[0]));
      }
      tmem_ld_wait();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&acc_empty[acc]);
    };
    auto store_sums = [&]() {
#pragma unroll
      for (int j = 0; j < BN; ++j)
        asm volatile("st.shared.f32 [%0], %1;" ::"r"(park + (uint32_t)((j * 128 + row) * 4)), "f"(sum[j]) : "memory");
    };
    if constexpr (kKind == Few::kDown) {
      int part = 0;
      for (int at = first; at < first + count; ++part) {
        const int unit = at / blocks;
        at = (unit + 1) * blocks;
        // Lane j: the weight of row j for this expert, and whether it is sent there.
        float factor = 0.f;
        bool sent = false;
        if (lane < p.m) {
          const int e = routing.used[unit];
          for (int j = 0; j < q.top_k; ++j) {
            if (routing.expert[lane * q.top_k + j] == e) {
              factor += routing.weight[lane * q.top_k + j];
              sent = true;
            }
          }
        }
        const uint32_t sent_rows = __ballot_sync(0xffffffffu, sent);
        float v[BN];
        take(part, v);
#pragma unroll
        for (int j = 0; j < BN; ++j) {
          const float f = __shfl_sync(0xffffffffu, factor, j);
          if ((sent_rows >> j) & 1u) sum[j] = fmaf(f, v[j], sum[j]);
        }
      }
    } else if (kKind == Few::kUp && split == 1) {
      for (int unit = 0; unit < units; ++unit) {
        take(unit, sum);
        store_sums();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (ok) finish_rows<BN, kKind, kGated, 1>(q, park, 0, rows, (long long)place_of(unit) * BN, tile_of(unit) * 64);
        asm volatile("bar.sync 1, 128;" ::: "memory");  // the sums may be written over
      }
    } else if (count > 0) {
      take(0, sum);
    }
    if (kKind != Few::kUp || split > 1) {
      // The ring is idle: every finishing warp has waited for the last MMA (one that gave up stores nothing).
      asm volatile("bar.sync 1, 128;" ::: "memory");
      if (kKind == Few::kDown) chain_wait();  // the residual and y belong to the kernels before as well
      if (kKind != Few::kDown || q.parts == nullptr) {
        store_sums();
      } else {
        // The last of a tile's parts to arrive adds them all up, its own as the others from memory.
        const int tile = (int)blockIdx.x, parts = split;
        float* own = q.parts + ((long long)(tile * parts + rank) * BN) * 128 + row;
#pragma unroll
        for (int j = 0; j < BN; ++j)
          if (j < rows) __stcg(own + j * 128, sum[j]);
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        int* flag = reinterpret_cast<int*>(park_at);
        if (threadIdx.x == 0) *flag = atomicAdd(&q.arrived[tile], 1);
        asm volatile("bar.sync 1, 128;" ::: "memory");
        const bool last = *flag == parts - 1;
        __threadfence();
        asm volatile("bar.sync 1, 128;" ::: "memory");
        if (last) {
#pragma unroll
          for (int j = 0; j < BN; ++j) sum[j] = 0.f;
          const float* from = q.parts + (long long)(tile * parts) * BN * 128 + row;
          // Several parts' loads in flight; added one after the other.
          constexpr int kAtOnce = BN <= 64 ? 64 / BN : 1;
          for (int part = 0; part < parts; part += kAtOnce) {
            float v[kAtOnce][BN];
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
              for (int j = 0; j < BN; ++j)
                v[u][j] = part + u < parts && j < rows ? __ldcg(from + ((long long)(part + u) * BN + j) * 128) : 0.f;
            }
#pragma unroll
            for (int u = 0; u < kAtOnce; ++u) {
#pragma unroll
              for (int j = 0; j < BN; ++j) sum[j] += v[u][j];
            }
          }
          store_sums();
          asm volatile("bar.sync 1, 128;" ::: "memory");
          if (ok) finish_rows<BN, kKind, kGated, 1>(q, park, 0, rows, 0, tile * 128);
        }
      }
    }
  }
  __syncwarp();
  cluster_sync_all();
  // kDown without an expert in use: the residual.
  if (warp < 4 && ok &&
      (kKind == Few::kDense || (kKind == Few::kUp && split > 1 && units > 0) || (kKind == Few::kDown && q.parts == nullptr))) {
    const long long to0 = kKind == Few::kUp ? (long long)place_of(0) * BN : row0;
    const int channel0 = tile_of(0) * (kGated ? 64 : 128);
    switch (split) {
      case 1: finish_rows<BN, kKind, kGated, 1>(q, park, rank, rows, to0, channel0); break;
      case 2: finish_rows<BN, kKind, kGated, 2>(q, park, rank, rows, to0, channel0); break;
      case 4: finish_rows<BN, kKind, kGated, 4>(q, park, rank, rows, to0, channel0); break;
      default: finish_rows<BN, kKind, kGated, 8>(q, park, rank, rows, to0, channel0); break;
    }
  }
  __syncwarp();
  cluster_sync_all();  // no CTA leaves while another may still read its sums
  tc_fence_before();
  __syncthreads();
  if (warp == 5) {
    tc_fence_after();
    tmem_dealloc(tmem, kTmemColumns);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Weight rows [experts][n or 2 n][k]; any row count.
inline int few_weight_map(CUtensorMap* out, const Product& p, int experts, int box_rows) {
  const uint64_t row = (uint64_t)p.ldw * 2;
  const uint64_t dims[3] = {(uint64_t)p.k, (uint64_t)p.n * (p.gated ? 2 : 1), (uint64_t)experts};
  const uint64_t strides[2] = {row, experts > 1 ? (uint64_t)p.w_expert * 2 : row};
  const uint32_t box[3] = {64, (uint32_t)box_rows, 1};
  return operand_map_bf16(out, 3, p.w, dims, strides, box);
}

template <int BN, Few kKind, bool kGated>
int launch_few(const CUtensorMap& map_w, const CUtensorMap& map_x, const FewParams& q, long long tiles, int split, int row_tiles,
               cudaStream_t stream) {
  using S = FewSmem<BN, kKind>;
  static bool configured[64] = {false};
  int dev = 0;
  MIE_CUDA(cudaGetDevice(&dev));
  if (dev >= 0 && dev < 64 && !configured[dev]) {
    MIE_CUDA(cudaFuncSetAttribute(product_few_kernel<BN, kKind, kGated>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  S::kTotal));
    configured[dev] = true;
  }
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)tiles, (unsigned)split, (unsigned)row_tiles);
  config.blockDim = dim3(kFewThreads, 1, 1);
  config.dynamicSmemBytes = S::kTotal;
  config.stream = stream;
  cudaLaunchAttribute attr[2];
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 1;
  attr[0].val.clusterDim.y = kKind == Few::kDown && q.parts != nullptr ? 1u : (unsigned)split;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = chained_launch_enabled() ? 2 : 1;
  prefer_shared_carveout(reinterpret_cast<const void*>(product_few_kernel<BN, kKind, kGated>));
  MIE_CUDA(cudaLaunchKernelEx(&config, product_few_kernel<BN, kKind, kGated>, map_w, map_x, q));
  MIE_LAUNCH_CHECK("product_few_kernel");
  return MIE_OK;
}

// CTAs a tile's K is cut over: as many, in powers of two, as surely run at once and have a few blocks each.
inline int few_split(long long tiles, int blocks, int ctas_per_sm) {
  const long long slots = (long long)ctas_per_sm * sm_count() * 9 / 10;
  int split = 1;
  while (split < 8 && tiles * split * 2 <= slots && blocks >= 4 * split) split *= 2;
  return split;
}

}  // namespace
}  // namespace mie
