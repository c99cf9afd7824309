// R2: general expert routing (scores, balance bias, groups, top-k) and its gradient.
//
// Forward, per token with logits l:
//   s_e   = exp(l_e - m) / sum_i exp(l_i - m)   or   1 / (1 + exp(-l_e));  an expert whose logit is
//           -inf or NaN is unavailable: it scores 0, stays out of the softmax and is never picked
//   key_e = l_e without a bias (both scores are monotone in it), s_e + b_e with one
//   groups: a group is worth its largest key, or the sum of its two largest s_e + b_e; the
//           topk_groups best stay open
//   picks:  the k largest keys of the open groups, every tie to the lower id; a slot no available
//           expert is left for gets id E and weight 0 (the expert kernels skip such ids)
//   w_j   = c r_j / sum_i r_i  or  c r_j,  with r_j the picked s (a zero sum gives zeros)
//
// The picks compare scores, and two scores that differ in their 9th digit have to come out in
// the order of their true values, so the keys are held in 64 bits.
//
// Backward, with g the gradient of w:
//   dr_j = c (g_j - sum_i g_i r_i / R) / R  (R = sum r)   or   c g_j
//   sigmoid: dl_e = dr_e s_e (1 - s_e);  softmax: dl_e = s_e (dr_e - sum_i dr_i r_i)
// The bias steers the picks only and has no gradient.
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace cmoe {

namespace {

constexpr int kWarps = 4;  // rows of a block, one per warp

__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  return v;
}
__device__ __forceinline__ float warp_max(float v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(0xffffffffu, v, o));
  return v;
}

// Largest key of the warp's lanes and its id, ties to the lower id.
__device__ __forceinline__ void warp_best(double& v, int& id) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const double ov = __shfl_xor_sync(0xffffffffu, v, o);
    const int oi = __shfl_xor_sync(0xffffffffu, id, o);
    if (ov > v || (ov == v && oi < id)) {
      v = ov;
      id = oi;
    }
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32) route_experts_kernel(RouteExpertsParams p) {
  extern __shared__ double smem_d[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  double* key = smem_d + warp * (2 * p.E + kRouteMaxGroups);
  double* sum_key = key + p.E;  // s + b, for the sums of two
  double* value = sum_key + p.E;
  const int per = p.E / p.num_groups;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp; row < p.num_tokens;
       row += static_cast<int64_t>(gridDim.x) * kWarps) {
    const T* l = static_cast<const T*>(p.logits) + row * p.stride;
    auto logit = [&](int e) {
      const float x = Elem<T>::to_f(l[e]);
      return x == x ? x : -CUDART_INF_F;
    };
    float m = -CUDART_INF_F;
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit(e));
    m = warp_max(m);
    double total = 0.0;
    if (p.scoring == 0) {
      for (int e = lane; e < p.E; e += 32) {
        const float x = logit(e);
        if (x > -CUDART_INF_F) total += exp(static_cast<double>(x) - static_cast<double>(m));
      }
      total = warp_sum(total);
    }
    auto score = [&](float x) -> double {
      if (!(x > -CUDART_INF_F)) return 0.0;
      if (p.scoring == 0) return exp(static_cast<double>(x) - static_cast<double>(m)) / total;
      return 1.0 / (1.0 + exp(-static_cast<double>(x)));
    };
    for (int e = lane; e < p.E; e += 32) {
      const float x = logit(e);
      double s = -CUDART_INF, k = -CUDART_INF;
      if (x > -CUDART_INF_F) {
        s = score(x) + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
        if (!(s > -CUDART_INF)) s = -CUDART_INF;  // a bias of -inf or NaN shuts the expert off
        k = p.bias ? s : static_cast<double>(x);
      }
      key[e] = k;
      sum_key[e] = s;
    }
    __syncwarp();
    if (p.num_groups > 1) {
      for (int g = lane; g < p.num_groups; g += 32) {
        double a = -CUDART_INF, b = -CUDART_INF;
        const double* from = p.group_score == 0 ? key : sum_key;
        for (int i = 0; i < per; ++i) {
          const double v = from[g * per + i];
          if (v > a) {
            b = a;
            a = v;
          } else if (v > b) {
            b = v;
          }
        }
        value[g] = (p.group_score == 0 || !(b > -CUDART_INF)) ? a : a + b;
      }
      __syncwarp();
      unsigned open = 0;
      for (int i = 0; i < p.topk_groups; ++i) {
        double v = -CUDART_INF;
        int id = 0x7fffffff;
        if (lane < p.num_groups && !((open >> lane) & 1u)) {
          v = value[lane];
          id = lane;
        }
        warp_best(v, id);
        if (!(v > -CUDART_INF)) break;
        open |= 1u << id;
      }
      for (int e = lane; e < p.E; e += 32)
        if (!((open >> (e / per)) & 1u)) key[e] = -CUDART_INF;
      __syncwarp();
    }
    float mine = 0.f;  // the pick of slot `lane`
    int mine_id = p.E;
    for (int j = 0; j < p.k; ++j) {
      double v = -CUDART_INF;
      int id = 0x7fffffff;
      for (int e = lane; e < p.E; e += 32)
        if (key[e] > v) {
          v = key[e];
          id = e;
        }
      warp_best(v, id);
      if (!(v > -CUDART_INF)) break;
      if (lane == j) {
        mine = static_cast<float>(score(logit(id)));
        mine_id = id;
      }
      if (id % 32 == lane) key[id] = -CUDART_INF;
      __syncwarp();
    }
    if (p.renormalize) {
      const float r = warp_sum(mine);
      mine = r > 0.f ? mine / r : mine;
    }
    if (lane < p.k) {
      p.weights[row * p.k + lane] = mine * p.scaling;
      p.indices[row * p.k + lane] = mine_id;
    }
    __syncwarp();
  }
}

template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    route_experts_backward_kernel(RouteExpertsBackwardParams p) {
  extern __shared__ float smem_f[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* ds = smem_f + warp * p.E;
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp; row < p.num_tokens;
       row += static_cast<int64_t>(gridDim.x) * kWarps) {
    const T* l = static_cast<const T*>(p.logits) + row * p.stride;
    T* out = static_cast<T*>(p.grad_logits) + row * p.E;
    auto logit = [&](int e) {
      const float x = Elem<T>::to_f(l[e]);
      return x == x ? x : -CUDART_INF_F;
    };
    float m = -CUDART_INF_F, total = 0.f;
    if (p.scoring == 0) {
      for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit(e));
      m = warp_max(m);
      for (int e = lane; e < p.E; e += 32)
        if (logit(e) > -CUDART_INF_F) total += expf(logit(e) - m);
      total = warp_sum(total);
    }
    auto score = [&](float x) -> float {
      if (!(x > -CUDART_INF_F)) return 0.f;
      return p.scoring == 0 ? expf(x - m) / total : 1.f / (1.f + expf(-x));
    };
    for (int e = lane; e < p.E; e += 32) ds[e] = 0.f;
    float g = 0.f, r = 0.f;
    int id = p.E;
    if (lane < p.k) {
      id = p.indices[row * p.k + lane];
      if (id >= 0 && id < p.E) {
        g = p.grad_weights[row * p.k + lane] * p.scaling;
        r = score(logit(id));
      } else {
        id = p.E;
      }
    }
    float dr = g;
    if (p.renormalize) {
      const float R = warp_sum(r);
      dr = R > 0.f ? (g - warp_sum(g * (r / R))) / R : 0.f;
    }
    const float D = p.scoring == 0 ? (p.renormalize ? 0.f : warp_sum(dr * r)) : 0.f;
    __syncwarp();
    for (int j = 0; j < p.k; ++j) {  // in slot order: one id twice adds up, always the same way
      if (lane == j && id < p.E) ds[id] += dr;
      __syncwarp();
    }
    for (int e = lane; e < p.E; e += 32) {
      const float s = score(logit(e));
      const float d = p.scoring == 0 ? s * (ds[e] - D) : ds[e] * s * (1.f - s);
      out[e] = Elem<T>::from_f(d);
    }
    __syncwarp();
  }
}

int blocks_for(int64_t rows, int num_sms) {
  const int64_t b = (rows + kWarps - 1) / kWarps, cap = static_cast<int64_t>(num_sms) * 8;
  return static_cast<int>(b < cap ? b : cap);
}

}  // namespace

int launch_route_experts(int dtype, const RouteExpertsParams& p, int num_sms, cudaStream_t s) {
  if (p.num_tokens <= 0) return 0;
  const int grid = blocks_for(p.num_tokens, num_sms);
  const size_t smem = sizeof(double) * kWarps * (2 * p.E + kRouteMaxGroups);
  if (dtype == kF32) route_experts_kernel<float><<<grid, kWarps * 32, smem, s>>>(p);
  else if (dtype == kBF16) route_experts_kernel<__nv_bfloat16><<<grid, kWarps * 32, smem, s>>>(p);
  else route_experts_kernel<__half><<<grid, kWarps * 32, smem, s>>>(p);
  return 0;
}

int launch_route_experts_backward(int dtype, const RouteExpertsBackwardParams& p, int num_sms,
                                  cudaStream_t s) {
  if (p.num_tokens <= 0) return 0;
  const int grid = blocks_for(p.num_tokens, num_sms);
  const size_t smem = sizeof(float) * kWarps * p.E;
  if (dtype == kF32) route_experts_backward_kernel<float><<<grid, kWarps * 32, smem, s>>>(p);
  else if (dtype == kBF16)
    route_experts_backward_kernel<__nv_bfloat16><<<grid, kWarps * 32, smem, s>>>(p);
  else route_experts_backward_kernel<__half><<<grid, kWarps * 32, smem, s>>>(p);
  return 0;
}

}  // namespace cmoe
