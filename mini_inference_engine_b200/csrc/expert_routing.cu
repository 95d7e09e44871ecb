// Routing of tokens to experts: scores, choice and weights from a router's logits.
//
//   s = softmax(z) or sigmoid(z) over a token's E logits,   c = s + b (c = s without a bias), -inf where z = -inf
//   groups: the top_groups groups whose group_best largest c add up to most stay in the choice
//   ids = the top_k experts by c, descending, equal ones by their index;   w = s[ids] (/ their sum) * scale
//
// A warp takes a token and keeps its logits in registers; a choice is one maximum over the warp (`redux.sync`) and one
// minimum over the indices that have it, so that equal values go to the lowest index.
//
// The choice is that of 64 bits.  Without a bias, and with groups judged by their best expert, the order of the scores is the
// order of the logits, which are compared as they are.  Otherwise c is computed in 32 bits with an error below 2^-20 (1 + |c|)
// (exponential 2 ulp, its argument's rounding, a sum of up to 1024 terms, a quotient, the bias' addition; each at most a few
// 2^-24 of a value in [0, 1] or of c).  Where two values that decide something are nearer than twice that and do not come
// from equal logits and biases, the warp decides the token again in 64 bits.
#include "common.cuh"

namespace mie {
namespace {

constexpr int kRouteWarps = 8;
constexpr float kUncertain = 1.9073486e-6f;  // 2^-19

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
  const uint32_t u = __float_as_uint(v == 0.f ? 0.f : v);  // -0 equals 0
  return v != v ? 1u : (u >> 31) ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float key_value(uint32_t k) {
  return k == 1u ? __uint_as_float(0x7fc00000u) : __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ unsigned long long order_key(double v) {
  const unsigned long long u = (unsigned long long)__double_as_longlong(v == 0.0 ? 0.0 : v);
  return v != v ? 1ull : (u >> 63) ? ~u : u | 0x8000000000000000ull;
}
__device__ __forceinline__ uint32_t warp_top(uint32_t key) { return __reduce_max_sync(0xffffffffu, key); }
__device__ __forceinline__ unsigned long long warp_top(unsigned long long key) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const unsigned long long other = __shfl_xor_sync(0xffffffffu, key, o);
    key = other > key ? other : key;
  }
  return key;
}
__device__ __forceinline__ bool far_apart(float a, float b, float size) { return fabsf(a - b) > kUncertain * (1.f + size); }

// A row's choice in 64 bits (see above), by the whole warp; `scratch` and `chosen` are shared memory of the warp.
template <typename T>
__device__ __noinline__ void choose_again(const RouteParams& p, const T* row, float top, double* scratch, int* chosen) {
  const int lane = threadIdx.x & 31, size = p.experts / p.groups;
  double sum = 0.0;
  if (!p.sigmoid) {
    for (int e = lane; e < p.experts; e += 32) sum += exp((double)to_float<T>(row[e]) - (double)top);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
  }
  for (int e = lane; e < p.experts; e += 32) {
    const double v = (double)to_float<T>(row[e]);
    double c = p.sigmoid ? 1.0 / (1.0 + exp(-v)) : exp(v - (double)top) / sum;
    if (p.bias != nullptr) c += (double)p.bias[e];
    scratch[e] = v == -(double)INFINITY ? v : c;
  }
  __syncwarp();
  uint32_t kept = 0xffffffffu;
  if (p.groups > 1) {
    unsigned long long mine = 0;
    if (lane < p.groups) {
      double first = -(double)INFINITY, second = first;
      bool bad = false;
      for (int i = 0; i < size; ++i) {
        const double c = scratch[lane * size + i];
        bad |= c != c;
        if (c > first) {
          second = first;
          first = c;
        } else if (c > second) {
          second = c;
        }
      }
      mine = bad ? 1ull : order_key(p.group_best == 2 ? first + second : first);
    }
    kept = 0;
    for (int j = 0; j < p.top_groups; ++j) {
      const unsigned long long best = warp_top(mine);
      const int g = (int)__reduce_min_sync(0xffffffffu, mine == best ? (uint32_t)lane : 32u);
      kept |= 1u << g;
      if (lane == g) mine = 0;
    }
  }
  for (int j = 0; j < p.top_k; ++j) {
    unsigned long long mine = 0;
    int at = 0;
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
    const unsigned long long best = warp_top(mine);
    const int e = (int)__reduce_min_sync(0xffffffffu, mine == best ? (uint32_t)at : 0x7fffffffu);
    if (lane == 0) chosen[j] = e;
    if ((e & 31) == lane) scratch[e] = __longlong_as_double(0x7ff8000000000001ll);
    __syncwarp();
  }
}

// Bound by HBM for many tokens (a logit is read once) and by the chain of maxima for few.
template <typename T, int V>
__global__ void __launch_bounds__(kRouteWarps * 32) route_kernel(const RouteParams p) {
  extern __shared__ double scratch_all[];  // groups or a bias: the row's c, [warp][32 V]
  __shared__ int chosen_all[kRouteWarps][32];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int size = p.experts / p.groups;
  const bool by_logit = p.bias == nullptr && (p.groups == 1 || p.group_best == 1);
  const bool whole_sum = !p.sigmoid && (!p.renormalize || !by_logit);
  double* scratch = scratch_all + warp * 32 * V;
  float* row_c = reinterpret_cast<float*>(scratch);
  int* chosen = chosen_all[warp];
  chain_release();
  chain_wait();
  for (long long t = (long long)blockIdx.x * kRouteWarps + warp; t < p.tokens; t += (long long)gridDim.x * kRouteWarps) {
    const T* row = reinterpret_cast<const T*>(p.logits) + t * p.ld;
    float z[V];
    uint32_t key[V];
    float top = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      z[i] = e < p.experts ? to_float<T>(row[e]) : -INFINITY;
      bad |= z[i] != z[i];
      top = fmaxf(top, z[i]);
    }
    bad = __any_sync(0xffffffffu, bad);
    top = warp_max(top);
    float sum = 0.f;
    if (whole_sum) {
#pragma unroll
      for (int i = 0; i < V; ++i) sum += z[i] == -INFINITY ? 0.f : expf(z[i] - top);
      sum = warp_sum(sum);
    }
    auto score = [&](float v) {
      if (v == -INFINITY) return 0.f;
      return p.sigmoid ? 1.f / (1.f + expf(-v)) : expf(v - top);  // softmax: not yet divided by the sum
    };
    bool sure = true;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int e = lane + 32 * i;
      float c = z[i];
      if (!by_logit && c != -INFINITY) {
        c = score(z[i]);
        if (!p.sigmoid) c = c / sum;
        if (p.bias != nullptr && e < p.experts) c += p.bias[e];
      }
      key[i] = e < p.experts ? order_key(c) : 0u;
      if (p.groups > 1 && e < p.experts) row_c[e] = c;
    }
    if (p.groups > 1) {
      __syncwarp();
      uint32_t mine = 0;
      float magnitude = 0.f;
      if (lane < p.groups) {
        float first = -INFINITY, second = first;
        bool nan = false;
        for (int i = 0; i < size; ++i) {
          const float c = row_c[lane * size + i];
          nan |= c != c;
          if (c > first) {
            second = first;
            first = c;
          } else if (c > second) {
            second = c;
          }
        }
        mine = nan ? 1u : order_key(p.group_best == 2 ? first + second : first);
        magnitude = fabsf(first) + (p.group_best == 2 ? fabsf(second) : 0.f);
      }
      uint32_t kept = 0, last = 0;
      float last_magnitude = 0.f;
      for (int j = 0; j <= p.top_groups && j < p.groups; ++j) {
        const uint32_t best = warp_top(mine);
        const int g = (int)__reduce_min_sync(0xffffffffu, mine == best ? (uint32_t)lane : 32u);
        const float size_now = __shfl_sync(0xffffffffu, magnitude, g);
        if (j == p.top_groups) {  // the first group left out has to be clearly behind the last one taken
          sure = by_logit || far_apart(key_value(last), key_value(best), 1.f + last_magnitude + size_now);
          break;
        }
        kept |= 1u << g;
        last = best;
        last_magnitude = size_now;
        if (lane == g) mine = 0;
      }
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const int e = lane + 32 * i;
        if (e < p.experts && !((kept >> (e / size)) & 1u)) key[i] = 0;
      }
      __syncwarp();
    }
    float my_score = 0.f, total = 0.f;  // lane j: the j-th choice
    uint32_t before = 0;
    float before_z = 0.f, before_b = 0.f;
    int my_id = 0;
    const int picks = by_logit ? p.top_k : p.top_k + 1;  // one more, to know how far it is behind
    for (int j = 0; j < picks && sure; ++j) {
      uint32_t mine = 0;
      int at = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (key[i] > mine) {
          mine = key[i];
          at = lane + 32 * i;
        }
      }
      const uint32_t best = warp_top(mine);
      if (best == 0) break;  // every expert has been taken
      const int e = (int)__reduce_min_sync(0xffffffffu, mine == best ? (uint32_t)at : 0x7fffffffu);
      float v = 0.f;
#pragma unroll
      for (int i = 0; i < V; ++i) {
        if (lane + 32 * i == e) {
          v = z[i];
          key[i] = 0;
        }
      }
      v = __shfl_sync(0xffffffffu, v, e & 31);
      if (!by_logit) {
        const float b = p.bias != nullptr ? p.bias[e] : 0.f;
        if (j > 0 && !(v == before_z && b == before_b) && !(v == -INFINITY && before_z == -INFINITY))
          sure = far_apart(key_value(before), key_value(best), fabsf(key_value(before)));
        before = best;
        before_z = v;
        before_b = b;
      }
      if (j < p.top_k && lane == j) {
        my_id = e;
        my_score = v;
      }
    }
    if (!sure) {
      choose_again<T>(p, row, top, scratch, chosen);
      if (lane < p.top_k) {
        my_id = chosen[lane];
        my_score = to_float<T>(row[my_id]);
      }
      __syncwarp();
    }
    my_score = lane < p.top_k ? score(my_score) : 0.f;
    total = p.renormalize ? warp_sum(my_score) : p.sigmoid ? 1.f : sum;
    if (lane < p.top_k) {
      const float w = total == 0.f ? 0.f : my_score / total;  // nothing to choose from
      p.ids[t * p.top_k + lane] = my_id;
      p.weights[t * p.top_k + lane] = bad ? __uint_as_float(0x7fc00000u) : w * p.scale;
    }
  }
}

template <typename T, int V>
int launch_route(const RouteParams& p, cudaStream_t stream) {
  const int smem = p.groups > 1 || p.bias != nullptr ? kRouteWarps * 32 * V * (int)sizeof(double) : 0;
  static bool configured[64] = {false};
  int dev = 0;
  MIE_CUDA(cudaGetDevice(&dev));
  if (V == 32 && dev >= 0 && dev < 64 && !configured[dev]) {
    MIE_CUDA(cudaFuncSetAttribute(route_kernel<T, V>, cudaFuncAttributeMaxDynamicSharedMemorySize, 64 * 1024));
    configured[dev] = true;
  }
  const long long blocks = ((long long)p.tokens + kRouteWarps - 1) / kRouteWarps, most = 8ll * sm_count();
  MIE_CUDA(launch_chained(route_kernel<T, V>, dim3((unsigned)(blocks < most ? blocks : most)), dim3(kRouteWarps * 32),
                          (size_t)smem, stream, p));
  MIE_LAUNCH_CHECK("route_kernel");
  return MIE_OK;
}

template <typename T>
int launch_route(const RouteParams& p, cudaStream_t stream) {
  if (p.experts <= 32) return launch_route<T, 1>(p, stream);
  if (p.experts <= 64) return launch_route<T, 2>(p, stream);
  if (p.experts <= 128) return launch_route<T, 4>(p, stream);
  if (p.experts <= 256) return launch_route<T, 8>(p, stream);
  if (p.experts <= 512) return launch_route<T, 16>(p, stream);
  return launch_route<T, 32>(p, stream);
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
