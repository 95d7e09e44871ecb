// Routing of tokens to experts: scores, choice and weights from a router's logits.
//
//   s = softmax(z) or sigmoid(z) over a token's E logits,   c = s + b (c = s without a bias), -inf where z = -inf
//   groups: the top_groups groups whose group_best largest c add up to most stay in the choice
//   ids = the top_k experts by c, descending, equal ones by their index;   w = s[ids] (/ their sum) * scale
//
// 8, 16 or 32 lanes take a token (32 / lanes of them a warp), runs of V experts a lane, so that the lowest lane that has the
// largest value has the lowest index.  Every lane sorts its run once; a choice is then one maximum over the token's lanes'
// heads, and the lane that has it moves on.  Little data and many dependent steps: bound by instruction issue for many tokens
// and by latency for few.  One token of 128 3.1 us, 30011 of 64 7.8, 4096 of 256 by groups and bias 16.4 (its bytes 0.7; a lane
// that scanned its run for every choice took 18.1 of the second, 39.5 of the third with whole rows decided again in 64 bits).
// With a bias, 4096 of 512 take 65 us and of 1024 260: the runs' 16 and 32 entries a lane fill the registers, 32 spill.
//
// Without a bias, and with one group or groups judged by their best expert, the order of the scores is the order of the logits,
// which are compared as they are.  Otherwise the choice is that of c in 64 bits (where large sigmoids may be equal whose logits
// are not).  c is computed in 32 bits with an error below 2^-19 (1 + |c|)
// (approximate exponential and reciprocal 2^-22 each, the argument's rounding, a sum of up to 1024 terms, the bias' addition,
// of a value in [0, 1] or of c).  Where two values that decide something are nearer than twice that and do not come from
// equal logits and biases, the choice goes on to whatever is as near, and those candidates are ordered by c in 64 bits (all
// experts, where there are more than 32).  Neighbours are compared down to the first one left out; where that one equals the
// last one taken, the others are looked through for one as near (has_rival; 4096 equal rows of 256 12.7 -> 24.1 us, rows without
// equals at the border within 1 %).  Groups that are as near are decided again first.
#include "common.cuh"
#include "glue.cuh"

namespace mie {
namespace {

constexpr int kRouteWarps = 4;
constexpr float kUncertain = 3.8146973e-6f;  // 2^-18
constexpr uint32_t kAll = 0xffffffffu;

struct RouteParams {
  const void* logits;
  long long ld;
  const float* bias;
  int sigmoid, tokens, experts, top_k, groups, top_groups, group_best, renormalize;
  float scale;
  int* ids;
  float* weights;
};

// Monotonic integers of floating values: above 1 for every number; NaN is 1, below -inf and above 0, "not to be chosen".
__device__ __forceinline__ uint32_t order_key(float v) {
  const uint32_t u = __float_as_uint(v + 0.f);  // -0 equals 0
  return v != v ? 1u : u ^ ((uint32_t)((int)u >> 31) | 0x80000000u);
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k <= 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v + 0.0);
  return v != v ? 1ull : (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ bool far_apart(float a, float b, float size) { return fabsf(a - b) > kUncertain * (1.f + size); }

// Over the L lanes of a token.
template <int L>
__device__ __forceinline__ float token_max(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
template <int L>
__device__ __forceinline__ float token_sum(float v) {
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v += __shfl_xor_sync(kAll, v, o);
  return v;
}
template <int L>
__device__ __forceinline__ uint32_t token_top(uint32_t v) {
  if constexpr (L == 32) return __reduce_max_sync(kAll, v);
#pragma unroll
  for (int o = L / 2; o > 0; o >>= 1) v = max(v, __shfl_xor_sync(kAll, v, o));
  return v;
}
// The token's lanes for which `yes`, lane 0 of the token in bit 0.
template <int L>
__device__ __forceinline__ uint32_t token_lanes(bool yes) {
  const uint32_t all = __ballot_sync(kAll, yes);
  return L == 32 ? all : (all >> ((threadIdx.x & 31) / L * L)) & ((1u << (L & 31)) - 1u);
}
// Largest two of two descending pairs.
__device__ __forceinline__ void merge_two(float& first, float& second, float a, float b) {
  second = fmaxf(fminf(first, a), fmaxf(second, b));
  first = fmaxf(first, a);
}

// A token's c in 64 bits to `scratch`, by a whole warp.
template <typename T>
__device__ __forceinline__ void scores_again(const RouteParams& p, const T* row, float top, double* scratch) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
#pragma unroll 4
  for (int e = lane; e < p.experts; e += 32) {
    const float z = to_float<T>(row[e]);
    const double s = exp(p.sigmoid ? -(double)z : (double)z - (double)top);
    sum += s;
    scratch[e] = s;
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
#pragma unroll 4
  for (int e = lane; e < p.experts; e += 32) {
    const double s = scratch[e];
    double c = p.sigmoid ? 1.0 / (1.0 + s) : s / sum;
    if (p.bias != nullptr) c += (double)p.bias[e];
    scratch[e] = to_float<T>(row[e]) == -INFINITY ? -(double)INFINITY : c;
  }
  __syncwarp();
}

// The groups that a token is chosen from, as bits, by their c in 64 bits.
template <typename T>
__device__ __noinline__ uint32_t choose_groups_again(const RouteParams& p, const T* row, float top, double* scratch) {
  const int lane = threadIdx.x & 31, size = p.experts / p.groups;
  scores_again<T>(p, row, top, scratch);
  int lanes = 32;  // of a group
  while (lanes * p.groups > 32) lanes >>= 1;
  const int group = lane / lanes;
  double first = -(double)INFINITY, second = first;
  int bad = 0;
  if (group < p.groups) {
    for (int i = lane % lanes; i < size; i += lanes) {
      const double c = scratch[group * size + i];
      bad |= c != c;
      if (c > first) {
        second = first;
        first = c;
      } else if (c > second) {
        second = c;
      }
    }
  }
  for (int o = 1; o < lanes; o <<= 1) {
    const double a = __shfl_xor_sync(kAll, first, o), b = __shfl_xor_sync(kAll, second, o);
    bad |= __shfl_xor_sync(kAll, bad, o);
    second = a > first ? (first > b ? first : b) : (second > a ? second : a);
    first = a > first ? a : first;
  }
  const unsigned long long mine = bad ? 1ull : order_key(p.group_best == 2 ? first + second : first);
  int rank = 0;
  for (int g = 0; g < p.groups; ++g) {
    const unsigned long long other = __shfl_sync(kAll, mine, g * lanes);
    rank += other > mine || (other == mine && g < group);
  }
  const bool taken = group < p.groups && lane % lanes == 0 && rank < p.top_groups;
  const uint32_t kept = __reduce_or_sync(kAll, taken ? 1u << group : 0u);
  __syncwarp();
  return kept;
}

// A token's choice from the groups `kept`, all in 64 bits.
template <typename T>
__device__ __noinline__ void choose_again(const RouteParams& p, const T* row, float top, uint32_t kept, double* scratch, int* ids) {
  const int lane = threadIdx.x & 31, size = p.experts / p.groups;
  scores_again<T>(p, row, top, scratch);
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long mine = 0;
    int at = 0x7fffffff;
    for (int e = lane; e < p.experts; e += 32) {
      if (!((kept >> (p.groups > 1 ? e / size : 0)) & 1u)) continue;
      const double c = scratch[e];
      // A choice already made is held as a NaN with its lowest bit set.
      const unsigned long long key = __double_as_longlong(c) == 0x7ff8000000000001ll ? 0ull : order_key(c);
      if (key > mine) {
        mine = key;
        at = e;
      }
    }
    unsigned long long best = mine;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) {
      const unsigned long long other = __shfl_xor_sync(kAll, best, o);
      best = other > best ? other : best;
    }
    const int e = (int)__reduce_min_sync(kAll, mine == best ? (uint32_t)at : 0x7fffffffu);
    if (lane == 0) ids[j] = e;
    if ((e & 31) == lane) scratch[e] = __longlong_as_double(0x7ff8000000000001ll);
    __syncwarp();
  }
}

// Orders the first `count` (at most 32) entries of `ids` by their c in 64 bits, by a whole warp; the first top_k are the choice.
template <typename T>
__device__ __noinline__ void order_candidates(const RouteParams& p, const T* row, float top, int count, int* ids) {
  const int lane = threadIdx.x & 31;
  double sum = 0.0;
  if (!p.sigmoid) {
#pragma unroll 4
    for (int e = lane; e < p.experts; e += 32) sum += exp((double)to_float<T>(row[e]) - (double)top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(kAll, sum, o);
  }
  const int e = lane < count ? ids[lane] : 0;
  unsigned long long mine = 0;
  if (lane < count) {
    const double z = (double)to_float<T>(row[e]);
    double c = p.sigmoid ? 1.0 / (1.0 + exp(-z)) : exp(z - (double)top) / sum;
    if (p.bias != nullptr) c += (double)p.bias[e];
    mine = order_key(z == -(double)INFINITY ? z : c);
  }
  int rank = 0;
  for (int j = 0; j < count; ++j) {
    const unsigned long long other = __shfl_sync(kAll, mine, j);
    const int other_e = __shfl_sync(kAll, e, j);
    rank += other > mine || (other == mine && other_e < e);
  }
  __syncwarp();
  if (lane < count) ids[rank] = e;
  __syncwarp();
}

// Equal in every number of bits: equal logits and biases, or both masked.
template <typename T>
__device__ __forceinline__ bool same_choice(const RouteParams& p, const T* row, int a, int b) {
  const float za = to_float<T>(row[a]), zb = to_float<T>(row[b]);
  return (za == zb && (p.bias == nullptr || p.bias[a] == p.bias[b])) || (za == -INFINITY && zb == -INFINITY);
}

// Whether the groups `kept` have an expert that 32 bits do not tell from `last` though it is another choice, by a whole warp.
// (These c and those that were compared are off by 2^-19 each: twice the distance.)
template <typename T>
__device__ __noinline__ bool has_rival(const RouteParams& p, const T* row, float top, float sum, uint32_t kept, int last) {
  const int lane = threadIdx.x & 31, size = p.experts / p.groups;
  auto choice = [&](int e) {
    const float z = to_float<T>(row[e]);
    if (z == -INFINITY) return z;
    return (p.sigmoid ? 1.f / (1.f + expf(-z)) : expf(z - top) / sum) + (p.bias != nullptr ? p.bias[e] : 0.f);
  };
  const float border = choice(last), near = 2.f * kUncertain * (1.f + fabsf(border));
  if (border == -INFINITY) return false;  // so is all that is left, in the order of the indices
  bool found = false;
#pragma unroll 1
  for (int e = lane; e < p.experts; e += 32) {
    if (!((kept >> (p.groups > 1 ? e / size : 0)) & 1u)) continue;
    found |= !(fabsf(border - choice(e)) > near) && !same_choice<T>(p, row, last, e);
  }
  return __any_sync(kAll, found);
}

// Descending by (key, low): Batcher's odd-even merge sort.
template <int V>
__device__ __forceinline__ void sort_run(uint32_t (&key)[V], uint32_t (&low)[V]) {
#pragma unroll
  for (int p = 1; p < V; p <<= 1) {
#pragma unroll
    for (int k = p; k >= 1; k >>= 1) {
#pragma unroll
      for (int j = k % p; j + k < V; j += 2 * k) {
#pragma unroll
        for (int i = 0; i < k; ++i) {
          if (i + j + k < V && (i + j) / (2 * p) == (i + j + k) / (2 * p)) {
            const int a = i + j, b = i + j + k;
            const bool swap = key[b] > key[a] || (key[b] == key[a] && low[b] > low[a]);
            const uint32_t ka = key[a], la = low[a];
            key[a] = swap ? key[b] : ka;
            low[a] = swap ? low[b] : la;
            key[b] = swap ? ka : key[b];
            low[b] = swap ? la : low[b];
          }
        }
      }
    }
  }
}

template <typename T, int L, int V, bool kByLogit>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  constexpr int kTokens = 32 / L;  // of a warp
  extern __shared__ double scratch_all[];  // groups or a bias: a row's c, [warp][L V]
  __shared__ int chosen_all[kRouteWarps][kTokens][32];
  __shared__ float group_all[kRouteWarps][kTokens][2][32];  // score, magnitude
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, own = lane / L, l = lane % L;
  const int size = p.experts / p.groups, e0 = l * V;
  const bool whole_sum = !p.sigmoid && (!p.renormalize || !kByLogit);
  // Groups of whole lanes, in a power of two of them, find their best by shuffles.
  const int group_lanes = size % V == 0 && ((size / V) & (size / V - 1)) == 0 ? size / V : 0;
  double* scratch = scratch_all + (p.groups > 1 || !kByLogit ? warp * L * V : 0);
  float* row_c = reinterpret_cast<float*>(scratch);
  int* chosen = chosen_all[warp][own];
  float *group_score = group_all[warp][own][0], *group_size = group_all[warp][own][1];
  chain_release();
  chain_wait();
  float bias[V];
  if (!kByLogit) {
#pragma unroll
    for (int i = 0; i < V; ++i) bias[i] = p.bias != nullptr && e0 + i < p.experts ? p.bias[e0 + i] : 0.f;
  }
  const bool vec = p.experts == L * V && p.ld * sizeof(T) % 16 == 0 && (reinterpret_cast<uintptr_t>(p.logits) & 15) == 0;
  const long long step = (long long)gridDim.x * kRouteWarps * kTokens;
  for (long long t0 = ((long long)blockIdx.x * kRouteWarps + warp) * kTokens; t0 < p.tokens; t0 += step) {
    const long long t = t0 + own < p.tokens ? t0 + own : p.tokens - 1;  // lanes without a token take the last one too
    const T* row = reinterpret_cast<const T*>(p.logits) + t * p.ld;
    float z[V];
    constexpr int kVec = 16 / (int)sizeof(T) < V ? 16 / (int)sizeof(T) : V;
    if (vec && kVec * sizeof(T) == 16) {
#pragma unroll
      for (int i = 0; i < V; i += kVec) {
        const uint4 raw = *reinterpret_cast<const uint4*>(row + e0 + i);
        const T* v = reinterpret_cast<const T*>(&raw);
#pragma unroll
        for (int j = 0; j < kVec; ++j) z[i + j] = to_float<T>(v[j]);
      }
    } else {
#pragma unroll
      for (int i = 0; i < V; ++i) z[i] = e0 + i < p.experts ? to_float<T>(row[e0 + i]) : -INFINITY;
    }
    bool bad = false;
    float top = -INFINITY;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      bad |= z[i] != z[i];
      top = fmaxf(top, z[i]);
    }
    bad = token_lanes<L>(bad) != 0;
    top = token_max<L>(top);
    float sum = 0.f;
    if (whole_sum) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum += z[i] == -INFINITY ? 0.f : expf(z[i] - top);
      sum = token_sum<L>(sum);
    }
    uint32_t key[V], low[V];
    uint32_t kept = kAll;
    if (!kByLogit) {
      // z is c from here on.
      if (p.sigmoid) {
#pragma unroll
        for (int i = 0; i < V; ++i)
          z[i] = z[i] == -INFINITY ? z[i] : gate_quotient(1.f, gate_denominator(z[i] * -kLog2e)) + bias[i];
      } else {
        const float over = 1.f / sum;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float e;
          asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(e) : "f"((z[i] - top) * kLog2e));
          z[i] = z[i] == -INFINITY ? z[i] : fmaf(e, over, bias[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) {
      key[i] = order_key(z[i]);
      low[i] = V - 1 - i;
    }
    if (p.groups > 1) {
      const bool two = p.group_best == 2;
      if (group_lanes > 0) {
        float first = -INFINITY, second = -INFINITY;
        bool nan = false;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          nan |= z[i] != z[i];
          second = fmaxf(second, fminf(first, z[i]));
          first = fmaxf(first, z[i]);
        }
        for (int o = 1; o < group_lanes; o <<= 1) {
          const float a = __shfl_xor_sync(kAll, first, o), b = __shfl_xor_sync(kAll, second, o);
          nan |= __shfl_xor_sync(kAll, (int)nan, o) != 0;
          merge_two(first, second, a, b);
        }
        if (l % group_lanes == 0 && l / group_lanes < p.groups) {
          group_score[l / group_lanes] = nan ? __uint_as_float(0x7fc00000u) : two ? first + second : first;
          group_size[l / group_lanes] = fabsf(first) + (two ? fabsf(second) : 0.f);
        }
      } else {
        // One token of the warp after the other through the shared row.
        for (int s = 0; s < kTokens; ++s) {
          if (own == s) {
#pragma unroll
            for (int i = 0; i < V; ++i)
              if (e0 + i < p.experts) row_c[e0 + i] = z[i];
          }
          __syncwarp();
          if (lane < p.groups) {
            float first = -INFINITY, second = first;
            bool nan = false;
            for (int i = 0; i < size; ++i) {
              const float c = row_c[lane * size + i];
              nan |= c != c;
              second = fmaxf(second, fminf(first, c));
              first = fmaxf(first, c);
            }
            group_all[warp][s][0][lane] = nan ? __uint_as_float(0x7fc00000u) : two ? first + second : first;
            group_all[warp][s][1][lane] = fabsf(first) + (two ? fabsf(second) : 0.f);
          }
          __syncwarp();
        }
      }
      __syncwarp();
      // Rank of every group; the last one taken and the first one left out have to be clearly apart.
      kept = 0;
      float border = INFINITY, border_size = 0.f, next = -INFINITY, next_size = 0.f;
      bool number = true;
      for (int g = l; g < p.groups; g += L) {
        const uint32_t k = order_key(group_score[g]);
        int rank = 0;
        for (int o = 0; o < p.groups; ++o) {
          const uint32_t other = order_key(group_score[o]);
          rank += other > k || (other == k && o < g);
        }
        if (rank < p.top_groups) kept |= 1u << g;
        number &= k > 1u;
        if (rank == p.top_groups - 1) border = group_score[g], border_size = group_size[g];
        if (rank == p.top_groups) next = group_score[g], next_size = group_size[g];
      }
#pragma unroll
      for (int o = L / 2; o > 0; o >>= 1) {
        kept |= __shfl_xor_sync(kAll, kept, o);
        if (!kByLogit) {
          border = fminf(border, __shfl_xor_sync(kAll, border, o));
          next = fmaxf(next, __shfl_xor_sync(kAll, next, o));
          border_size = fmaxf(border_size, __shfl_xor_sync(kAll, border_size, o));
          next_size = fmaxf(next_size, __shfl_xor_sync(kAll, next_size, o));
        }
      }
      if (!kByLogit && p.top_groups < p.groups) {
        const bool sure = token_lanes<L>(!number) == 0 && far_apart(border, next, 1.f + border_size + next_size);
        uint32_t again = __ballot_sync(kAll, !sure);
        __syncwarp();
        while (again != 0) {
          const int s = (__ffs(again) - 1) / L, from = s * L;
          again &= ~((L == 32 ? kAll : (1u << (L & 31)) - 1u) << from);
          const T* which = reinterpret_cast<const T*>(p.logits) + __shfl_sync(kAll, t, from) * p.ld;
          const uint32_t theirs = choose_groups_again<T>(p, which, __shfl_sync(kAll, top, from), scratch);
          if (own == s) kept = theirs;
        }
      }
      // V consecutive experts are of one or a few groups.
      int g = e0 / size, left = size - (e0 - g * size);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (left == 0) {
          ++g;
          left = size;
        }
        --left;
        if (e0 + i < p.experts && !((kept >> g) & 1u)) key[i] = 0;
      }
      __syncwarp();
    }
    if (e0 + V > p.experts) {
#pragma unroll
      for (int i = 0; i < V; ++i)
        if (e0 + i >= p.experts) key[i] = 0;
    }
    sort_run(key, low);
    // The largest head of the token's lanes; the first lane that has it moves on.
    auto take = [&](uint32_t& best) {
      best = token_top<L>(key[0]);
      const int first = __ffs(token_lanes<L>(key[0] == best)) - 1;
      const int e = e0 + V - 1 - (int)low[0];
      if (l == first) {
#pragma unroll
        for (int i = 0; i + 1 < V; ++i) {
          key[i] = key[i + 1];
          low[i] = low[i + 1];
        }
        key[V - 1] = 0;
      }
      return L == 32 && kByLogit ? (l == first ? e : -1) : __shfl_sync(kAll, e, own * L + first);
    };
    if constexpr (kByLogit) {
      for (int j = 0; j < p.top_k; ++j) {
        uint32_t best;
        const int e = take(best);
        if (L == 32 ? e >= 0 : l == 0) chosen[j] = e;
      }
    } else {
      uint32_t last = 0;
      int last_e = 0, count = 0;
      bool near_ties = false, equal_border = false;  // the last expert taken and the first one left out
      float least = INFINITY;  // candidates are not below it
      for (int j = 0; j <= p.top_k || (j < 32 && __any_sync(kAll, near_ties && count == j)); ++j) {
        uint32_t best;
        const int e = take(best);
        if (l == 0 && j < 32) chosen[j] = e;
        if (best == 0) continue;  // every expert has been taken
        const float value = key_value(best);
        if (j > 0 && j <= p.top_k) {
          const float a = key_value(last);
          if (!far_apart(a, value, fabsf(a))) {
            const bool same = same_choice<T>(p, row, last_e, e);
            near_ties |= !same;
            equal_border = same && j == p.top_k;
          }
        }
        if (j == p.top_k - 1) least = value - 2.f * kUncertain * (1.f + fabsf(value));
        if (count == j && (j < p.top_k || value >= least)) count = j + 1;
        last = best;
        last_e = e;
      }
      // More candidates than are held, or values that are no numbers: all over again.
      bool all_again = near_ties && (count >= 32 || !(least == least));
      __syncwarp();
      // Behind equals at the border there may be others as near, which no comparison of neighbours has seen.
      uint32_t ask = __ballot_sync(kAll, equal_border && !near_ties);
      while (ask != 0) {
        const int s = (__ffs(ask) - 1) / L, from = s * L;
        ask &= ~((L == 32 ? kAll : (1u << (L & 31)) - 1u) << from);
        const T* which = reinterpret_cast<const T*>(p.logits) + __shfl_sync(kAll, t, from) * p.ld;
        const bool rival = has_rival<T>(p, which, __shfl_sync(kAll, top, from), __shfl_sync(kAll, sum, from),
                                        __shfl_sync(kAll, kept, from), chosen_all[warp][s][p.top_k - 1]);
        if (own == s && rival) near_ties = all_again = true;
      }
      uint32_t again = __ballot_sync(kAll, near_ties);
      __syncwarp();
      while (again != 0) {
        const int s = (__ffs(again) - 1) / L, from = s * L;
        again &= ~((L == 32 ? kAll : (1u << (L & 31)) - 1u) << from);
        const T* which = reinterpret_cast<const T*>(p.logits) + __shfl_sync(kAll, t, from) * p.ld;
        const float its_top = __shfl_sync(kAll, top, from);
        const int candidates = __shfl_sync(kAll, count, from);
        if (__shfl_sync(kAll, (int)all_again, from))
          choose_again<T>(p, which, its_top, __shfl_sync(kAll, kept, from), scratch, chosen_all[warp][s]);
        else
          order_candidates<T>(p, which, its_top, candidates, chosen_all[warp][s]);
      }
    }
    __syncwarp();
    // Over the chosen's sum only their ratios count.  So exponentials are taken against the largest of the chosen, which may be
    // far below the row's; a sigmoid is exp(z) / (1 + exp(z)), and of it the numerator as long as the largest is below 0.
    float total = p.sigmoid ? 1.f : sum, shift = p.sigmoid ? 0.f : top;
    if (p.renormalize) {
      shift = -INFINITY;
      for (int j = l; j < p.top_k; j += L) shift = fmaxf(shift, to_float<T>(row[chosen[j]]));
      shift = token_max<L>(shift);
      if (p.sigmoid) shift = fminf(shift, 0.f);
    }
    auto weight = [&](float v) {
      if (v == -INFINITY) return 0.f;
      if (!p.sigmoid) return expf(v - shift);
      return v > 0.f ? 1.f / (1.f + expf(-v)) : expf(v - shift) / (1.f + expf(v));
    };
    if (p.renormalize) {
      total = 0.f;
      for (int j = l; j < p.top_k; j += L) total += weight(to_float<T>(row[chosen[j]]));
      total = token_sum<L>(total);
    }
    if (t0 + own < p.tokens) {
      for (int j = l; j < p.top_k; j += L) {
        const int e = chosen[j];
        const float s = weight(to_float<T>(row[e]));
        const float w = total == 0.f ? 0.f : s / total;  // nothing to choose from
        p.ids[t * p.top_k + j] = e;
        p.weights[t * p.top_k + j] = bad ? __uint_as_float(0x7fc00000u) : w * p.scale;
      }
    }
    __syncwarp();  // `chosen` is used again
  }
}

template <typename T, int L, int V, bool kByLogit>
int launch_route(const RouteParams& p, cudaStream_t stream) {
  const int smem = p.groups > 1 || !kByLogit ? kRouteWarps * L * V * (int)sizeof(double) : 0;
  const int per_block = kRouteWarps * (32 / L);
  const long long blocks = ((long long)p.tokens + per_block - 1) / per_block, most = 16ll * sm_count();
  MIE_CUDA(launch_chained(route_kernel<T, L, V, kByLogit>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kRouteWarps * 32),
                          (size_t)smem, stream, p));
  MIE_LAUNCH_CHECK("route_kernel");
  return MIE_OK;
}

template <typename T, bool kByLogit>
int launch_route(const RouteParams& p, cudaStream_t stream) {
  if (p.experts <= 32) return launch_route<T, 8, 4, kByLogit>(p, stream);
  if (p.experts <= 64) return launch_route<T, 8, 8, kByLogit>(p, stream);
  if (p.experts <= 128) return launch_route<T, 16, 8, kByLogit>(p, stream);
  if (p.experts <= 256) return launch_route<T, 32, 8, kByLogit>(p, stream);
  if (p.experts <= 512) return launch_route<T, 32, 16, kByLogit>(p, stream);
  return launch_route<T, 32, 32, kByLogit>(p, stream);
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t stream) {
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_best == 1);
  return by_logit ? launch_route<T, true>(p, stream) : launch_route<T, false>(p, stream);
}

}  // namespace
}  // namespace mie

using namespace mie;

extern "C" int mie_route_experts(const void* logits, int64_t ld, int32_t dtype, const float* bias, int32_t scores,
                                 int32_t tokens, int32_t experts, int32_t top_k, int32_t groups, int32_t top_groups,
                                 int32_t group_best, int32_t renormalize, float scale, int32_t* ids, float* weights,
                                 void* stream_) {
  cudaStream_t stream = (cudaStream_t)stream_;
  MIE_CHECK_ARG(logits && ids && weights, "null pointer");
  MIE_CHECK_ARG(dtype >= MIE_DTYPE_BF16 && dtype <= MIE_DTYPE_F32, "logits are bf16, fp16 or fp32");
  MIE_CHECK_ARG(tokens >= 0 && experts >= 1 && experts <= MIE_MAX_EXPERTS && ld >= experts, "invalid sizes: %d tokens, %d experts",
                tokens, experts);
  MIE_CHECK_ARG(scores == MIE_SCORES_SOFTMAX || scores == MIE_SCORES_SIGMOID, "unknown scores %d", scores);
  MIE_CHECK_ARG(groups >= 1 && groups <= 32 && experts % groups == 0 && top_groups >= 1 && top_groups <= groups,
                "%d experts cannot be chosen from %d of %d groups", experts, top_groups, groups);
  MIE_CHECK_ARG(group_best >= 1 && group_best <= 2 && group_best <= experts / groups, "groups are judged by their best one or two");
  MIE_CHECK_ARG(top_k >= 1 && top_k <= MIE_MAX_TOP_K && top_k <= top_groups * (experts / groups),
                "cannot choose %d experts from %d groups of %d", top_k, top_groups, experts / groups);
  if (tokens == 0) return MIE_OK;
  const RouteParams p{logits, ld, bias, scores == MIE_SCORES_SIGMOID, tokens, experts, top_k, groups, top_groups,
                      group_best, renormalize != 0, scale, ids, weights};
  if (dtype == MIE_DTYPE_F32) return launch_route<float>(p, stream);
  if (dtype == MIE_DTYPE_F16) return launch_route<__half>(p, stream);
  return launch_route<__nv_bfloat16>(p, stream);
}
