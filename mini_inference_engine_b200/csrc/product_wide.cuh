// Products of many rows on CTA pairs.
//
// A pair (`cta_group::2`) multiplies 256 weight rows, 128 of each CTA, with up to 256 rows of x, half of which each CTA
// stages: the weight rows are the M of the tensor-memory accumulator, the rows of x its N, so that a tile of few rows (the
// end of an expert's) takes a multiple of 16 columns' time and not 256.  Two accumulators: the epilogue of a tile runs under
// the products of the next.  One warp requests operands by 128-byte-swizzled TMA tiles, eight more those rows of x that are
// scattered (`tile::gather4`), one issues the MMAs of the pair, eight finish.
//
// What bounds it.  A block of 64 columns is 512 clocks of products at 256 rows, and 64 KB of operands a pair, 64 bytes a clock
// and SM: the products and L2 are about even, and under the power cap both.  8192 x 12288 x 4096 takes 536 us (1.54 PFLOP/s) in
// a burst and 620 to 640 back to back (1.3, at the clocks that 1000 W allow), the gate_up product of 65536 routed rows 304 us
// (1.36).  Smaller tiles load more per product: they are taken where fewer rounds or a fuller GPU are worth it (the caller's
// plan).  What else cost time on the way: gathers issued by one warp (75 to 90 clocks a request: 902 us with one warp, 455
// with four, 337 with eight and the rows' numbers in uniform registers, 308 apart from the weights' loads); handing an
// accumulator back with a release, which waits for the rows stored before (264 -> 207 us of down product); activations one by
// one (190 clocks each); finished values through shared memory, whose bandwidth the MMAs' operands take.
//
// So finished values go to y straight from the accumulator where they can (kDirect): the weight rows of a run of 32 are staged
// in the order 4 s + j -> 8 j + s, and a thread's four accumulators of a row of x (fragments 16 x 256b: lanes l / 4 and l / 4 + 8
// of either half) are neighbours in y.  Gated weights are staged as runs of 8 gates and 8 ups, a thread has a gate and its up,
// and the values go through shared memory, transposed by `stmatrix`, to whole runs of y's rows, as they do where y's rows are
// not whole runs of four.
//
// Where a product has fewer tiles than pairs, the K of a tile may be cut over the pairs of a cluster (kDense, kDirect), which
// park their sums in the idle ring and each finish a part of the rows.
#pragma once

#include "products.cuh"
#include "umma.cuh"

namespace mie {
namespace {

enum class Rows {
  kDense,  // y rows as x rows, bias, activation or gate, residual
  kUp,     // routed, gated: x gathered by pair, hidden rows in sorted order with the pair's weight
  kDown    // routed: sorted hidden rows, y rows in the same order as scaled fp16
};

// Finished values go to y straight from the accumulator's fragments (kDirect), or through shared memory.
template <bool kDirect>
constexpr int wide_stages() {
  return kDirect ? 7 : 6;
}
constexpr int kWideRows = 256;                 // rows of x a tile
constexpr int kWideStageBytes = 32 * 1024;     // 128 weight rows and up to 128 rows of x, 64 columns
constexpr int kWideFinishers = 8;              // warps
constexpr int kGatherers = 8;                  // warps that request gathered rows
template <Rows kRows>
constexpr int wide_threads() {
  return (kWideFinishers + 2 + (kRows == Rows::kUp ? kGatherers : 0)) * 32;
}
constexpr int kChunk = 32;                     // rows of x that are finished together
constexpr int kChunkBytes = kChunk * 256;
template <bool kDirect>
constexpr int wide_smem() {
  return wide_stages<kDirect>() * (kWideStageBytes + 16) + (kDirect ? 0 : 4 * kChunkBytes) + 4 * 8 + 16 + 1024;
}
static_assert(wide_smem<false>() <= 227 * 1024 && wide_smem<true>() <= 227 * 1024, "shared memory of an SM");

// A CTA's 128 weight rows as the finishers want them: gated, 8 runs of 8 gates and their 8 ups; direct, 4 runs of 32 in the
// order 4 s + j -> 8 j + s; otherwise as they are.  `all` brings them at once; where the last run is cut short they come run by
// run, the whole ones by `run`, the rest of the last one by `rest`.
struct WeightMaps {
  CUtensorMap all, run, rest;
};

struct WideParams {
  Product p;
  int row_tiles, tile_rows;  // kDense
  int weight_tiles, band;
  int x_box;                 // rows of x a TMA request brings (not gathered)
  int8_t* exponents;         // kDown: [pairs][exponent_ld], one per 32 channels
  int exponent_ld;
};

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(cols) : "memory");
}
__device__ __forceinline__ void tmem_relinquish_pair() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols) : "memory");
}
// Signals the barrier at this address in both CTAs of the pair whose first has cluster rank `leader`.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar, uint32_t leader) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                   smem_u32(bar)),
               "h"((uint16_t)(3u << leader))
               : "memory");
}
__device__ __forceinline__ void umma_f16_pair(uint32_t tmem_d, uint64_t desc_a, uint64_t desc_b, uint32_t idesc,
                                              uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
      :
      : "r"(tmem_d), "l"(desc_a), "l"(desc_b), "r"(idesc), "r"(accumulate)
      : "memory");
}
__device__ __forceinline__ uint32_t at_rank(const void* local, uint32_t rank) {
  uint32_t remote;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(remote) : "r"(smem_u32(local)), "r"(rank));
  return remote;
}
// Relaxed: tensor memory has been read when this is reached, and a release would wait for the rows stored before.
__device__ __forceinline__ void mbar_arrive_at(uint32_t cluster_addr) {
  asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
// TMA loads of this GPU's memory into this CTA, completing on a barrier of either CTA of the pair.
__device__ __forceinline__ void tma_pair_2d(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4}], [%2];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1)
      : "memory");
}
__device__ __forceinline__ void tma_pair_3d(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5}], "
      "[%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tma_pair_5d(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2, int c3,
                                            int c4) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, %4, %5, "
      "%6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4)
      : "memory");
}
// Four rows of 128 bytes.
__device__ __forceinline__ void tma_pair_gather4(void* dst, const CUtensorMap* map, uint32_t bar, int c0, int4 r) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cluster.global.tile::gather4.mbarrier::complete_tx::bytes.cta_group::2 [%0], [%1, {%3, "
      "%4, %5, %6, %7}], [%2];" ::"r"(smem_u32(dst)),
      "l"(map), "r"(bar), "r"(c0), "r"(r.x), "r"(r.y), "r"(r.z), "r"(r.w)
      : "memory");
}
// 16 lanes x 32 columns: lane l gets, for every run of 8 columns, columns 2 (l % 4) and + 1 of lanes l / 4 and l / 4 + 8.
__device__ __forceinline__ void tmem_ld_fragments(uint32_t addr, float (&v)[16]) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void stmatrix_x4_trans(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("stmatrix.sync.aligned.m8n8.x4.trans.shared.b16 [%0], {%1, %2, %3, %4};" ::"r"(addr), "r"(a), "r"(b), "r"(c),
               "r"(d)
               : "memory");
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) { return Mma16816<__nv_bfloat16>::pack(lo, hi); }

// Tile `index` of the launch.
struct WideTile {
  int expert, first, count, weight;
};
template <Rows kRows>
__device__ __forceinline__ WideTile wide_tile(const WideParams& q, int index) {
  if constexpr (kRows == Rows::kDense) {
    // Bands of row tiles go through all weights: what runs at one time shares both in L2.
    const int per_band = q.band * q.weight_tiles, band = index / per_band, in_band = index - band * per_band;
    const int wide = q.row_tiles - band * q.band < q.band ? q.row_tiles - band * q.band : q.band;
    const int weight = in_band / wide, row = band * q.band + in_band - weight * wide;
    const int first = row * q.tile_rows, left = q.p.m - first;
    return {0, first, left < q.tile_rows ? left : q.tile_rows, weight};
  } else {
    const int tile = index / q.weight_tiles;
    const RowTile t = q.p.tiles[tile];
    return {t.expert, t.first, t.count, index - tile * q.weight_tiles};
  }
}

// Where a finishing warp parks four of the 32 sums that a lane has of a chunk.
__device__ __forceinline__ int parked(int warp, int chunk, int four, int lane) {
  return ((warp * 4 + chunk) * 8 + four) * 512 + lane * 16;
}
static_assert(kWideFinishers * 4 * 8 * 512 <= wide_stages<true>() * kWideStageBytes, "the ring parks a tile's sums");

template <Rows kRows, bool kGated, bool kDirect>
__global__ void __launch_bounds__(wide_threads<kRows>(), 1)
    product_wide_kernel(const __grid_constant__ WeightMaps maps, const __grid_constant__ CUtensorMap map_x, const WideParams q) {
  static_assert(!(kGated && kDirect) && (kRows != Rows::kDown || kDirect), "what there are finishers for");
  constexpr int kWideStages = wide_stages<kDirect>();
  constexpr bool kSplits = kRows == Rows::kDense && kDirect;
  extern __shared__ uint8_t smem_raw[];
  uint8_t* ring = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~(uintptr_t)1023);
  uint8_t* chunks = ring + kWideStages * kWideStageBytes;  // [2 groups][2][kChunk][256], not kDirect
  uint64_t* full_bar = reinterpret_cast<uint64_t*>(chunks + (kDirect ? 0 : 4 * kChunkBytes));  // the first CTA's is used
  uint64_t* empty_bar = full_bar + kWideStages;
  uint64_t* acc_full = empty_bar + kWideStages;
  uint64_t* acc_empty = acc_full + 2;  // the first CTA's is used
  uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(acc_empty + 2);
  const Product& p = q.p;
  const int warp = uniform_warp_index(), lane = threadIdx.x & 31;
  // grid = (2 pairs, parts), cluster = (2, parts): the pairs of a cluster share the K of one tile.
  const int rank = blockIdx.x & 1, pair = blockIdx.x >> 1, pairs = gridDim.x >> 1;
  const int part = kSplits ? (int)blockIdx.y : 0, parts = kSplits ? (int)gridDim.y : 1;
  const uint32_t leader = 2u * (uint32_t)part;  // cluster rank of the pair's first CTA
  const int all_blocks = (p.k + 63) / 64, block0 = (int)((long long)all_blocks * part / parts);
  const int blocks = (int)((long long)all_blocks * (part + 1) / parts) - block0;

  if (warp == kWideFinishers && lane == 0) {
    for (int s = 0; s < kWideStages; ++s) {
      mbar_init(&full_bar[s], 1);
      mbar_init(&empty_bar[s], 1);
    }
    for (int a = 0; a < 2; ++a) {
      mbar_init(&acc_full[a], 1);
      mbar_init(&acc_empty[a], 2 * kWideFinishers);
    }
    mbar_fence_init();
    tma_prefetch_desc(&maps.all);
    tma_prefetch_desc(&map_x);
  }
  if (warp == kWideFinishers + 1) {
    tmem_alloc_pair(tmem_slot, 512);
    tmem_relinquish_pair();
  }
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();
  tc_fence_after();
  const uint32_t tmem = *tmem_slot;
  chain_release();
  chain_wait();
  const int tiles = (kRows == Rows::kDense ? q.row_tiles : *p.tile_count) * q.weight_tiles;

  if (warp == kWideFinishers) {
    int step = 0;
    bool ok = true;
    WideTile next = pair < tiles ? wide_tile<kRows>(q, pair) : WideTile{};
    for (int index = pair; index < tiles && ok; index += pairs) {
      const WideTile t = next;
      if (index + pairs < tiles) next = wide_tile<kRows>(q, index + pairs);  // read ahead of its use
      const int half = (t.count + 15) / 16 * 8;  // rows of x that a CTA stages
      const int boxes = kRows == Rows::kUp ? 0 : (half + q.x_box - 1) / q.x_box;
      const uint32_t bytes = 2u * (16384u + 128u * (uint32_t)(kRows == Rows::kUp ? half : boxes * q.x_box));
      const int first = t.first + rank * half;
      for (int b = 0; b < blocks; ++b, ++step) {
        const int s = step % kWideStages;
        uint8_t* dst = ring + (size_t)s * kWideStageBytes;
        if (!warp_wait_bounded(&empty_bar[s], ((step / kWideStages) & 1u) ^ 1u)) {
          raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t bar = at_rank(&full_bar[s], leader);
          if (rank == 0) mbar_expect_tx(&full_bar[s], bytes);
          if constexpr (kGated || kDirect) {
            constexpr int kRun = kGated ? 8 : 32, kRuns = kGated ? 8 : 4, kRunBytes = 16384 / kRuns;
            const int run = (t.weight * 2 + rank) * kRuns, whole = p.n / kRun;
            if (run + kRuns <= whole || whole * kRun == p.n) {
              tma_pair_5d(dst, &maps.all, bar, (block0 + b) * 64, 0, 0, run, t.expert);
            } else {
              for (int i = 0; i < kRuns; ++i) {
                if (run + i == whole)
                  tma_pair_5d(dst + i * kRunBytes, &maps.rest, bar, (block0 + b) * 64, 0, 0, 0, t.expert);
                else
                  tma_pair_5d(dst + i * kRunBytes, &maps.run, bar, (block0 + b) * 64, 0, 0, run + i, t.expert);
              }
            }
          } else {
            tma_pair_3d(dst, &maps.all, bar, (block0 + b) * 64, t.weight * 256 + rank * 128, t.expert);
          }
          for (int i = 0; i < boxes; ++i)
            tma_pair_2d(dst + 16384 + (size_t)i * q.x_box * 128, &map_x, bar, (block0 + b) * 64, first + i * q.x_box);
        }
        __syncwarp();
      }
    }
    // Every stage is free before this CTA ends: no signal of the other one is still under way to it.
    for (int i = 0; i < kWideStages && ok; ++i, ++step)
      ok = step < kWideStages || warp_wait_bounded(&empty_bar[step % kWideStages], ((step / kWideStages) & 1u) ^ 1u);
  } else if (kRows == Rows::kUp && warp > kWideFinishers + 1) {
    // Rows of x by fours: one request costs its warp about 75 clocks, so that several warps share a stage's 32.
    constexpr int kFours = 32 / kGatherers;
    const int gatherer = warp - kWideFinishers - 2;
    int step = 0, source = 0;
    bool ok = true;
    WideTile next = {};
    auto look_ahead = [&](int index) {  // the next tile and its rows, ahead of their use
      if (index >= tiles) return;
      next = wide_tile<kRows>(q, index);
      int row = rank * ((next.count + 15) / 16 * 8) + (lane / 4 * kGatherers + gatherer) * 4 + lane % 4;
      row = row < next.count ? row : next.count - 1;  // padding rows: any
      source = p.source[next.first + row];
    };
    look_ahead(pair);
    for (int index = pair; index < tiles && ok; index += pairs) {
      const int half = (next.count + 15) / 16 * 8;
      const int mine = (half / 4 - gatherer + kGatherers - 1) / kGatherers;  // fours of this warp
      const int row = source / p.source_divisor;
      int4 fours[kFours];
#pragma unroll
      for (int i = 0; i < kFours; ++i)
        fours[i] = make_int4(__shfl_sync(0xffffffffu, row, 4 * i), __shfl_sync(0xffffffffu, row, 4 * i + 1),
                             __shfl_sync(0xffffffffu, row, 4 * i + 2), __shfl_sync(0xffffffffu, row, 4 * i + 3));
      look_ahead(index + pairs);
      for (int b = 0; b < blocks; ++b, ++step) {
        const int s = step % kWideStages;
        if (!warp_wait_bounded(&empty_bar[s], ((step / kWideStages) & 1u) ^ 1u)) {
          raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
          ok = false;
          break;
        }
        if (elect_one()) {
          const uint32_t bar = at_rank(&full_bar[s], leader);
          uint8_t* dst = ring + (size_t)s * kWideStageBytes + 16384 + gatherer * 512;
#pragma unroll
          for (int i = 0; i < kFours; ++i)
            if (i < mine) tma_pair_gather4(dst + i * (kGatherers * 512), &map_x, bar, b * 64, fours[i]);
        }
        __syncwarp();
      }
    }
  } else if (warp == kWideFinishers + 1) {
    if (rank == 0) {
      int step = 0, round = 0;
      bool ok = true;
      WideTile next = pair < tiles ? wide_tile<kRows>(q, pair) : WideTile{};
      for (int index = pair; index < tiles && ok; index += pairs, ++round) {
        const WideTile t = next;
        if (index + pairs < tiles) next = wide_tile<kRows>(q, index + pairs);  // read ahead of its use
        const int acc = round & 1;
        if (!warp_wait_bounded(&acc_empty[acc], ((round >> 1) & 1u) ^ 1u)) {
          raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
          break;
        }
        tc_fence_after();
        const uint32_t idesc = instr_desc_bf16(256, (t.count + 15) / 16 * 16, 0, 0);
        for (int b = 0; b < blocks; ++b, ++step) {
          const int s = step % kWideStages;
          if (!warp_wait_bounded(&full_bar[s], (step / kWideStages) & 1u)) {
            raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
            ok = false;
            break;
          }
          tc_fence_after();
          if (elect_one()) {
            const uint32_t a = smem_u32(ring + (size_t)s * kWideStageBytes);
            const uint64_t da = smem_desc_k128(a), db = smem_desc_k128(a + 16384);
#pragma unroll
            for (int k = 0; k < 4; ++k)
              umma_f16_pair(tmem + acc * 256, da + (uint64_t)(2 * k), db + (uint64_t)(2 * k), idesc, b > 0 || k > 0 ? 1u : 0u);
            umma_commit_pair(&empty_bar[s], leader);
            if (b == blocks - 1) umma_commit_pair(&acc_full[acc], leader);
          }
          __syncwarp();
        }
      }
    }
  } else if constexpr (kDirect) {
    // 8 bytes a thread, 64 a row of y and warp.
    const int group = warp >> 2, quad = warp & 3, sub = lane >> 2, pick = lane & 3;
    int round = 0;
    bool ok = true;  // once a wait ran out nothing is stored
    for (int index = pair; index < tiles; index += pairs, ++round) {
      const WideTile t = wide_tile<kRows>(q, index);
      const int acc = round & 1;
      const int channel = t.weight * 256 + rank * 128 + quad * 32 + 4 * sub;  // the first of this thread's
      const int n_chunks = (t.count + kChunk - 1) / kChunk;
      const bool in = channel < p.n;
      float bias[4] = {0.f, 0.f, 0.f, 0.f};
      if (kRows == Rows::kDense && p.bias != nullptr && in) {
#pragma unroll
        for (int j = 0; j < 4; ++j) bias[j] = __bfloat162float(p.bias[channel + j]);
      }
      const bool has_residual = kRows == Rows::kDense && p.residual != nullptr;
      uint2 held[8];  // residual of the next chunk: rows 8 i + 2 pick + c
      auto load_residual = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const int row = chunk * kChunk + (i >> 1) * 8 + 2 * pick + (i & 1);
          held[i] = make_uint2(0, 0);
          if (row < t.count && in)
            held[i] = *reinterpret_cast<const uint2*>(p.residual + (long long)(t.first + row) * p.ldr + channel);
        }
      };
      auto finish = [&](int chunk, float (&v)[2][16]) {  // [j / 2][4 i + 2 (j % 2) + c]
        const int row0 = chunk * kChunk + 2 * pick;
        uint16_t* y = reinterpret_cast<uint16_t*>(p.y) + (long long)(t.first + row0) * p.ldy + channel;
        if constexpr (kRows == Rows::kDown) {
          // fp16 with an exponent per token and 32 channels: its largest finite value comes to lie in [2^14, 2^15).  Of the
          // largest only the exponent is needed, two tokens' to a word.
          uint32_t top[4];
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float a[2];
#pragma unroll
            for (int c = 0; c < 2; ++c)
              a[c] = fmaxf(fmaxf(fabsf(v[0][4 * i + c]), fabsf(v[0][4 * i + 2 + c])),
                           fmaxf(fabsf(v[1][4 * i + c]), fabsf(v[1][4 * i + 2 + c])));
            top[i] = (__float_as_uint(a[0]) >> 23) | (__float_as_uint(a[1]) >> 23 << 16);
          }
          bool infinite = false;
#pragma unroll
          for (int i = 0; i < 4; ++i) infinite |= (top[i] & 0xffffu) == 255u || (top[i] >> 16) == 255u;
          if (infinite) {  // by finite values alone
#pragma unroll
            for (int i = 0; i < 4; ++i) {
              top[i] = 0;
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                uint32_t most = 0;
#pragma unroll
                for (int m = 0; m < 4; ++m) {
                  const uint32_t e = __float_as_uint(v[m >> 1][4 * i + 2 * (m & 1) + c]) >> 23 & 255u;
                  most = e < 255u && e > most ? e : most;
                }
                top[i] |= most << (16 * c);
              }
            }
          }
#pragma unroll
          for (int o = 4; o < 32; o <<= 1) {
#pragma unroll
            for (int i = 0; i < 4; ++i) top[i] = __vmaxu2(top[i], __shfl_xor_sync(0xffffffffu, top[i], o));
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            // 2^(141 - e) as long as that is a normal number (e >= 15).
            const int e[2] = {max((int)(top[i] & 0xffffu), 15), max((int)(top[i] >> 16), 15)};
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              const float scale = __uint_as_float((uint32_t)(268 - e[c]) << 23);
              const uint2 out = make_uint2(Mma16816<__half>::pack(v[0][4 * i + c] * scale, v[0][4 * i + 2 + c] * scale),
                                           Mma16816<__half>::pack(v[1][4 * i + c] * scale, v[1][4 * i + 2 + c] * scale));
              if (row0 + 8 * i + c < t.count && in && ok) {
                *reinterpret_cast<uint2*>(y + (long long)(8 * i + c) * p.ldy) = out;
                if (sub == 0)
                  q.exponents[(long long)(t.first + row0 + 8 * i + c) * q.exponent_ld + channel / 32] = (int8_t)(141 - e[c]);
              }
            }
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int f = 0; f < 16; ++f) v[h][f] += bias[2 * h + ((f >> 1) & 1)];
            activate_all(p.activation, v[h]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              float a[4] = {v[0][4 * i + c], v[0][4 * i + 2 + c], v[1][4 * i + c], v[1][4 * i + 2 + c]};
              if (has_residual) {
                const float2 lo = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&held[2 * i + c].x));
                const float2 hi = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&held[2 * i + c].y));
                a[0] += lo.x, a[1] += lo.y, a[2] += hi.x, a[3] += hi.y;
              }
              if (row0 + 8 * i + c < t.count && in && ok)
                *reinterpret_cast<uint2*>(y + (long long)(8 * i + c) * p.ldy) =
                    make_uint2(pack_bf16(a[0], a[1]), pack_bf16(a[2], a[3]));
            }
          }
        }
      };
      const bool splits = kSplits && parts > 1;  // one tile a cluster
      if (has_residual && !splits && group < n_chunks) load_residual(group);
      if (ok && !warp_wait_bounded(&acc_full[acc], (round >> 1) & 1u)) {
        ok = false;
        raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
      }
      tc_fence_after();
      for (int chunk = group; chunk < n_chunks; chunk += 2) {
        float v[2][16];
        const uint32_t from = tmem + (uint32_t)(acc * 256 + chunk * kChunk) + ((uint32_t)(quad * 32) << 16);
        tmem_ld_fragments(from, v[0]);
        tmem_ld_fragments(from + (16u << 16), v[1]);
        tmem_ld_wait();
        if (chunk + 2 >= n_chunks) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_at(at_rank(&acc_empty[acc], leader));
        }
        if (splits) {
          // The ring is idle: this pair's last MMA is done.
#pragma unroll
          for (int i = 0; i < 8; ++i)
            *reinterpret_cast<float4*>(ring + parked(warp, chunk >> 1, i, lane)) =
                make_float4(v[i >> 2][4 * (i & 3)], v[i >> 2][4 * (i & 3) + 1], v[i >> 2][4 * (i & 3) + 2],
                            v[i >> 2][4 * (i & 3) + 3]);
        } else {
          finish(chunk, v);
          if (has_residual && chunk + 2 < n_chunks) load_residual(chunk + 2);
        }
      }
      if (group >= n_chunks) {  // no chunk of this tile
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(at_rank(&acc_empty[acc], leader));
      }
      if (splits) {
        // Every part finishes some of the chunks: the sums of all, in the order of the parts.
        __syncwarp();
        cluster_sync_all();
        for (int chunk = group + 2 * part; chunk < n_chunks; chunk += 2 * parts) {
          if (has_residual) load_residual(chunk);
          float v[2][16];
#pragma unroll
          for (int f = 0; f < 32; ++f) v[f >> 4][f & 15] = 0.f;
          for (int other = 0; other < parts; ++other) {
            float4 a[8];
#pragma unroll
            for (int i = 0; i < 8; ++i)
              a[i] = ld_cluster_f4(smem_u32(ring + parked(warp, chunk >> 1, i, lane)), 2u * (uint32_t)other + (uint32_t)rank);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
              v[i >> 2][4 * (i & 3)] += a[i].x;
              v[i >> 2][4 * (i & 3) + 1] += a[i].y;
              v[i >> 2][4 * (i & 3) + 2] += a[i].z;
              v[i >> 2][4 * (i & 3) + 3] += a[i].w;
            }
          }
          finish(chunk, v);
        }
      }
    }
  } else {
    constexpr int kCtaChannels = kGated ? 64 : 128;  // of y
    constexpr int kRowBytes = kCtaChannels * 2;
    const int group = warp >> 2, quad = warp & 3, threads_of_group = 128;
    const int sub = lane >> 2, pick = lane & 3;
    int round = 0, turn = 0;
    bool ok = true;  // once a wait ran out nothing is stored, but every barrier is met
    for (int index = pair; index < tiles; index += pairs, ++round) {
      const WideTile t = wide_tile<kRows>(q, index);
      const int acc = round & 1;
      const int channel0 = t.weight * (2 * kCtaChannels) + rank * kCtaChannels;
      const int n_chunks = (t.count + kChunk - 1) / kChunk;
      // Bias of this thread's channels.
      float bias[2][2] = {{0.f, 0.f}, {0.f, 0.f}};
      if (kRows == Rows::kDense && p.bias != nullptr) {
#pragma unroll
        for (int h = 0; h < 2; ++h) {
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            const int c = channel0 + (kGated ? quad * 16 + h * 8 + sub : quad * 32 + h * 16 + r * 8 + sub);
            if (c < p.n) bias[h][r] = __bfloat162float(p.bias[kGated && r ? p.n + c : c]);
          }
        }
      }
      const bool has_residual = kRows == Rows::kDense && p.residual != nullptr;
      constexpr int kLanesPerRow = kRowBytes / 16, kRowsPerStep = 128 / kLanesPerRow;
      const int store_row = (int)(threadIdx.x & 127) / kLanesPerRow, store_part = (int)(threadIdx.x & 127) % kLanesPerRow;
      const int store_channel = channel0 + store_part * 8;
      const bool vec_store = p.ldy % 8 == 0 && p.n % 8 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 15) == 0;
      const bool vec_residual = has_residual && p.ldr % 8 == 0 && (reinterpret_cast<uintptr_t>(p.residual) & 15) == 0;
      uint4 held[kChunk / kRowsPerStep];
      auto load_residual = [&](int chunk) {
#pragma unroll
        for (int i = 0; i < kChunk / kRowsPerStep; ++i) {
          const int row = chunk * kChunk + i * kRowsPerStep + store_row;
          held[i] = make_uint4(0, 0, 0, 0);
          if (row >= t.count || store_channel >= p.n) continue;
          const __nv_bfloat16* src = p.residual + (long long)(t.first + row) * p.ldr + store_channel;
          if (vec_residual && store_channel + 8 <= p.n) {
            held[i] = *reinterpret_cast<const uint4*>(src);
          } else {
            uint16_t e[8];
#pragma unroll
            for (int j = 0; j < 8; ++j)
              e[j] = store_channel + j < p.n ? reinterpret_cast<const uint16_t*>(src)[j] : (uint16_t)0;
            held[i] = make_uint4(e[0] | (uint32_t)e[1] << 16, e[2] | (uint32_t)e[3] << 16, e[4] | (uint32_t)e[5] << 16,
                                 e[6] | (uint32_t)e[7] << 16);
          }
        }
      };
      if (has_residual && group < n_chunks) load_residual(group);
      // Factor of the row that this lane knows of each of the group's chunks: read here, not between the stores.
      float factors[kWideRows / kChunk / 2];
      if (kRows == Rows::kUp) {
#pragma unroll
        for (int i = 0; i < kWideRows / kChunk / 2; ++i) {
          const int row = (group + 2 * i) * kChunk + lane;
          factors[i] = row < t.count ? p.factor[p.source[t.first + row]] : 0.f;
        }
      }
      if (ok && !warp_wait_bounded(&acc_full[acc], (round >> 1) & 1u)) {
        ok = false;
        raise_status(p.status, MIE_STATUS_WAIT_TIMEOUT);
      }
      tc_fence_after();
      bool released = false;
#pragma unroll
      for (int mine = 0; mine < kWideRows / kChunk / 2; ++mine) {
        const int chunk = group + 2 * mine;
        if (chunk >= n_chunks) break;
        ++turn;
        const float factor = kRows == Rows::kUp ? factors[mine] : 1.f;
        const int buffer = group * 2 + (turn & 1);
        uint8_t* stage = chunks + buffer * kChunkBytes;
        const uint32_t stage_addr = smem_u32(stage);
        float v[2][16];
        const uint32_t from = tmem + (uint32_t)(acc * 256 + chunk * kChunk) + ((uint32_t)(quad * 32) << 16);
        tmem_ld_fragments(from, v[0]);
        tmem_ld_fragments(from + (16u << 16), v[1]);
        tmem_ld_wait();
        if (chunk + 2 >= n_chunks) {
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive_at(at_rank(&acc_empty[acc], leader));
          released = true;
        }
        if (has_residual) {
#pragma unroll
          for (int i = 0; i < kChunk / kRowsPerStep; ++i) {
            const int row = i * kRowsPerStep + store_row;
            *reinterpret_cast<uint4*>(stage + row * kRowBytes + ((store_part ^ (row & 7)) * 16)) = held[i];
          }
          asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads_of_group) : "memory");
          if (chunk + 2 < n_chunks) load_residual(chunk + 2);
        }
        // Eight tokens at a time: matrices of 8 channels x 8 tokens, transposed on their way to [token][channel].
        const int part = lane >> 3, line = lane & 7;
        if constexpr (kGated) {
          float y[16];  // [8 tokens][h][2]
#pragma unroll
          for (int i = 0; i < 4; ++i) {
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              y[4 * i + 2 * h] = v[h][4 * i] + bias[h][0];
              y[4 * i + 2 * h + 1] = v[h][4 * i + 1] + bias[h][0];
            }
          }
          activate_all(p.activation, y);
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const float f0 = kRows == Rows::kUp ? __shfl_sync(0xffffffffu, factor, i * 8 + pick * 2) : 1.f;
            const float f1 = kRows == Rows::kUp ? __shfl_sync(0xffffffffu, factor, i * 8 + pick * 2 + 1) : 1.f;
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              y[4 * i + 2 * h] *= v[h][4 * i + 2] + bias[h][1];
              y[4 * i + 2 * h + 1] *= v[h][4 * i + 3] + bias[h][1];
              if (kRows == Rows::kUp) {
                y[4 * i + 2 * h] *= f0;
                y[4 * i + 2 * h + 1] *= f1;
              }
            }
          }
#pragma unroll
          for (int i = 0; i < 4; i += 2) {
            const int row = (i + (part >> 1)) * 8 + line;
            const uint32_t at = stage_addr + (uint32_t)(row * kRowBytes + (((quad * 2 + (part & 1)) ^ (row & 7)) * 16));
            if (has_residual) {
              uint32_t res[4];
              ldmatrix_x4_trans(res[0], res[1], res[2], res[3], at);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const float2 r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&res[m]));
                y[4 * i + 2 * m] += r.x;
                y[4 * i + 2 * m + 1] += r.y;
              }
            }
            stmatrix_x4_trans(at, pack_bf16(y[4 * i], y[4 * i + 1]), pack_bf16(y[4 * i + 2], y[4 * i + 3]),
                              pack_bf16(y[4 * i + 4], y[4 * i + 5]), pack_bf16(y[4 * i + 6], y[4 * i + 7]));
          }
        } else {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
#pragma unroll
            for (int f = 0; f < 16; ++f) v[h][f] += bias[h][(f >> 1) & 1];
            activate_all(p.activation, v[h]);
          }
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            const int row = i * 8 + line;
            const uint32_t at = stage_addr + (uint32_t)(row * kRowBytes + (((quad * 4 + part) ^ (row & 7)) * 16));
            if (has_residual) {
              uint32_t res[4];
              ldmatrix_x4_trans(res[0], res[1], res[2], res[3], at);
#pragma unroll
              for (int m = 0; m < 4; ++m) {
                const float2 r = __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&res[m]));
                v[m >> 1][4 * i + 2 * (m & 1)] += r.x;
                v[m >> 1][4 * i + 2 * (m & 1) + 1] += r.y;
              }
            }
            stmatrix_x4_trans(at, pack_bf16(v[0][4 * i], v[0][4 * i + 1]), pack_bf16(v[0][4 * i + 2], v[0][4 * i + 3]),
                              pack_bf16(v[1][4 * i], v[1][4 * i + 1]), pack_bf16(v[1][4 * i + 2], v[1][4 * i + 3]));
          }
        }
        asm volatile("bar.sync %0, %1;" ::"r"(1 + group), "r"(threads_of_group) : "memory");
        // Whole runs of y's rows.  The other buffer takes the next chunk, so that one barrier a chunk is enough.
        if (vec_store) {
          uint4 data[kChunk / kRowsPerStep];
#pragma unroll
          for (int i = 0; i < kChunk / kRowsPerStep; ++i) {
            const int row = i * kRowsPerStep + store_row;
            data[i] = *reinterpret_cast<const uint4*>(stage + row * kRowBytes + ((store_part ^ (row & 7)) * 16));
          }
#pragma unroll
          for (int i = 0; i < kChunk / kRowsPerStep; ++i) {
            const int row = chunk * kChunk + i * kRowsPerStep + store_row;
            if (row < t.count && ok && store_channel < p.n)
              *reinterpret_cast<uint4*>(reinterpret_cast<uint16_t*>(p.y) + (long long)(t.first + row) * p.ldy + store_channel) =
                  data[i];
          }
        } else {
          // Rows of any alignment: a warp takes eight of them, a lane whole words of y, the ends by halves.  (Eight halves a
          // lane, as its 16 bytes hold them, touch every sector of a row eight times.)
          constexpr int kWords = kCtaChannels / 64, kEach = kChunk / 4;
          const int valid = p.n - channel0 < kCtaChannels ? p.n - channel0 : kCtaChannels;
          uint32_t word[kEach][kWords];
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              const int row = quad * kEach + i, c = 2 * (lane + 32 * w);
              word[i][w] =
                  *reinterpret_cast<const uint32_t*>(stage + row * kRowBytes + (((c >> 3) ^ (row & 7)) * 16) + (c & 7) * 2);
            }
          }
#pragma unroll
          for (int i = 0; i < kEach; ++i) {
            const int row = chunk * kChunk + quad * kEach + i;
            uint16_t* dst = reinterpret_cast<uint16_t*>(p.y) + (long long)(t.first + row) * p.ldy + channel0;
            const int odd = (int)(reinterpret_cast<uintptr_t>(dst) >> 1 & 1);  // words of y begin at the next half
            const bool in = row < t.count && ok;
#pragma unroll
            for (int w = 0; w < kWords; ++w) {
              const int c = 2 * (lane + 32 * w) + odd;
              uint32_t v = word[i][w];
              if (odd) {  // the same for the whole warp
                if (w == 0 && lane == 0 && in && valid > 0) dst[0] = (uint16_t)v;
                uint32_t next = __shfl_down_sync(0xffffffffu, v, 1);
                const uint32_t wrapped = __shfl_sync(0xffffffffu, word[i][w + 1 < kWords ? w + 1 : w], 0);
                if (lane == 31) next = w + 1 < kWords ? wrapped : 0u;
                v = v >> 16 | next << 16;
              }
              if (!in) continue;
              if (c + 1 < valid)
                *reinterpret_cast<uint32_t*>(dst + c) = v;
              else if (c < valid)
                dst[c] = (uint16_t)v;
            }
          }
        }
      }
      if (!released) {  // a group without a chunk of this tile
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive_at(at_rank(&acc_empty[acc], leader));
      }
    }
  }
  __syncwarp();
  if (kSplits && parts > 1 && warp >= kWideFinishers) cluster_sync_all();  // the finishing warps' barrier before they add up
  tc_fence_before();
  __syncthreads();
  cluster_sync_all();  // no CTA leaves while its barriers or staged rows may be used by the other
  if (warp == kWideFinishers + 1) {
    tc_fence_after();
    tmem_dealloc_pair(tmem, 512);
  }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
inline bool rows_fit_tma(const void* ptr, long long stride) {
  return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0 && stride % 8 == 0;
}

inline int weight_maps(WeightMaps* out, const Product& p, int experts, bool direct) {
  const uint64_t row = (uint64_t)p.ldw * 2, expert = experts > 1 ? (uint64_t)p.w_expert * 2 : row, k = (uint64_t)p.k;
  if (!p.gated && !direct) {
    const uint64_t dims[3] = {k, (uint64_t)p.n, (uint64_t)experts};
    const uint64_t strides[2] = {row, expert};
    const uint32_t box[3] = {64, 128, 1};
    return operand_map_bf16(&out->all, 3, p.w, dims, strides, box);
  }
  // Runs: [8 rows][gate, up] or [8 rows 4 apart][4 rows].
  const uint32_t inner = p.gated ? 2 : 4, runs = p.gated ? 8 : 4;
  const int run = p.gated ? 8 : 32, whole = p.n / run, rest = p.n - whole * run;
  const uint64_t strides[4] = {p.gated ? row : 4 * row, p.gated ? (uint64_t)p.n * row : row, (uint64_t)run * row, expert};
  const uint32_t box[5] = {64, 8, inner, runs, 1}, one[5] = {64, 8, inner, 1, 1};
  const uint64_t dims[5] = {k, 8, inner, (uint64_t)(whole > 0 ? whole : 1), (uint64_t)experts};
  // A weight of less than a run has no whole one; what stands in its place is never loaded.
  const uint64_t rest_rows = (uint64_t)(p.gated ? rest : rest / 4);
  const uint64_t rest_dims[5] = {k, rest > 0 ? rest_rows : 8, inner, 1, (uint64_t)experts};
  const __nv_bfloat16* rest_base = rest > 0 ? p.w + (long long)whole * run * p.ldw : p.w;
  if (int rc = operand_map_bf16(&out->all, 5, p.w, dims, strides, box)) return rc;
  if (int rc = operand_map_bf16(&out->run, 5, p.w, dims, strides, one)) return rc;
  return operand_map_bf16(&out->rest, 5, rest_base, rest_dims, strides, one);
}
inline int row_map(CUtensorMap* out, const Product& p, long long rows, int box_rows) {
  const uint64_t dims[2] = {(uint64_t)p.k, (uint64_t)rows};
  const uint64_t strides[1] = {(uint64_t)p.ldx * 2};
  const uint32_t box[2] = {64, (uint32_t)box_rows};
  return operand_map_bf16(out, 2, p.x, dims, strides, box);
}
// What the pair kernel's loads ask of the operands.
inline bool wide_takes(const Product& p) {
  return p.k % 8 == 0 && rows_fit_tma(p.x, p.ldx) && rows_fit_tma(p.w, p.ldw) && p.w_expert % 8 == 0;
}

// Whether finished values may go to y (and come from the residual) by runs of four.
inline bool direct_takes(const Product& p) {
  return !p.gated && p.n % 4 == 0 && p.ldy % 4 == 0 && (reinterpret_cast<uintptr_t>(p.y) & 7) == 0 &&
         (p.residual == nullptr || (p.ldr % 4 == 0 && (reinterpret_cast<uintptr_t>(p.residual) & 7) == 0));
}

template <Rows kRows, bool kGated, bool kDirect>
cudaLaunchConfig_t wide_config(cudaLaunchAttribute (&attr)[2], int pairs, int parts, cudaStream_t stream) {
  cudaLaunchConfig_t config = {};
  config.gridDim = dim3((unsigned)(2 * pairs), (unsigned)parts);
  config.blockDim = dim3(wide_threads<kRows>());
  config.dynamicSmemBytes = wide_smem<kDirect>();
  config.stream = stream;
  attr[0].id = cudaLaunchAttributeClusterDimension;
  attr[0].val.clusterDim.x = 2;
  attr[0].val.clusterDim.y = (unsigned)parts;
  attr[0].val.clusterDim.z = 1;
  attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[1].val.programmaticStreamSerializationAllowed = 1;
  config.attrs = attr;
  config.numAttrs = chained_launch_enabled() ? 2 : 1;
  return config;
}

template <Rows kRows, bool kGated, bool kDirect>
int configure_wide() {
  static bool configured[64] = {false};
  int dev = 0;
  MIE_CUDA(cudaGetDevice(&dev));
  if (dev < 0 || dev >= 64 || !configured[dev]) {
    MIE_CUDA(cudaFuncSetAttribute(product_wide_kernel<kRows, kGated, kDirect>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                  wide_smem<kDirect>()));
    if (dev >= 0 && dev < 64) configured[dev] = true;
  }
  return MIE_OK;
}

// `parts` pairs share a tile's K (kDense, kDirect); then there are as many tiles as pairs.
template <Rows kRows, bool kGated, bool kDirect>
int launch_wide(const WeightMaps& maps, const CUtensorMap& map_x, const WideParams& q, long long most_tiles, int parts,
                cudaStream_t stream) {
  if (int rc = configure_wide<kRows, kGated, kDirect>()) return rc;
  const long long most = parts > 1 ? most_tiles : sm_count() / 2;
  cudaLaunchAttribute attr[2];
  const cudaLaunchConfig_t config =
      wide_config<kRows, kGated, kDirect>(attr, (int)(most_tiles < most ? most_tiles : most), parts, stream);
  prefer_shared_carveout(reinterpret_cast<const void*>(product_wide_kernel<kRows, kGated, kDirect>));
  MIE_CUDA(cudaLaunchKernelEx(&config, product_wide_kernel<kRows, kGated, kDirect>, maps, map_x, q));
  MIE_LAUNCH_CHECK("product_wide_kernel");
  return MIE_OK;
}

}  // namespace
}  // namespace mie
