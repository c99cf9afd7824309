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
// the order of their true values: a 32-bit comparison that its rounding errors could have
// turned is made again in 64 bits.
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

constexpr int kWarps = 4;      // rows of a block, one per warp
constexpr int kFastWarps = 8;  // the same for route_experts_kernel
constexpr int kMaxCand = 64;   // candidates it ranks

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

// NaN logits count as -inf.
template <typename T> __device__ __forceinline__ float logit_of(const T* l, int e) {
  const float x = Elem<T>::to_f(l[e]);
  return x == x ? x : -CUDART_INF_F;
}

// Doubles of scratch per warp of route_row64.
__host__ __device__ __forceinline__ int row64_scratch(int E) { return E; }

// Order-preserving map of doubles (no NaN) to unsigned 64-bit keys above 0.
__device__ __forceinline__ uint64_t order_key64(double v) {
  const uint64_t b = static_cast<uint64_t>(__double_as_longlong(v + 0.0));  // -0 as +0
  return (b >> 63) ? ~b : (b | (1ull << 63));
}

// A score in 64 bits.  One copy of the code (and loops that are not unrolled) in what follows:
// these paths run for a row in thousands, and what they cost then is fetching instructions.
__device__ __noinline__ double score64(float x, float m, double total, int scoring) {
  const double e = exp(scoring == 0 ? static_cast<double>(x) - static_cast<double>(m)
                                    : -static_cast<double>(x));
  return scoring == 0 ? e / total : 1.0 / (1.0 + e);
}

// One row by one warp with 64-bit keys, any shape; key: E doubles of scratch.  Leaves the pick of
// slot `lane` (id E: none) and its score.
template <typename T>
__device__ __noinline__ void route_row64(const RouteExpertsParams& p, int64_t row, double* key,
                                         float& mine, int& mine_id) {
  const int lane = threadIdx.x & 31;
  const T* l = static_cast<const T*>(p.logits) + row * p.stride;
  float m = -CUDART_INF_F;
  double total = 1.0;
  if (p.scoring == 0) {
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit_of(l, e));
    m = warp_max(m);
    double sum = 0.0;
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) {
      const float x = logit_of(l, e);
      sum += x > -CUDART_INF_F ? score64(x, m, 1.0, 0) : 0.0;
    }
    total = warp_sum(sum);
  }
  const bool sums = p.num_groups > 1 && p.group_score != 0;
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    const float x = logit_of(l, e);
    double k = static_cast<double>(x);
    if (p.bias || sums) {
      k = score64(x, m, total, p.scoring) + (p.bias ? static_cast<double>(p.bias[e]) : 0.0);
      // a bias of -inf or NaN shuts the expert off
      if (!(x > -CUDART_INF_F && k > -CUDART_INF)) k = -CUDART_INF;
    }
    key[e] = k;
  }
  __syncwarp();
  unsigned open = 0xffffffffu;
  const int per = p.E / p.num_groups;
  if (p.num_groups > 1) {
    const int lpg = 32 / p.num_groups, g = lane / lpg, at = lane % lpg;
    double a = -CUDART_INF, b = -CUDART_INF;
    if (g < p.num_groups) {
#pragma unroll 1
      for (int i = at; i < per; i += lpg) {
        const double v = key[g * per + i];
        b = fmax(b, fmin(a, v));
        a = fmax(a, v);
      }
    }
    double ga = a, gb = b;
#pragma unroll 1
    for (int o = 1; o < lpg; ++o) {
      const int from = (g * lpg + (at + o) % lpg) & 31;
      const double oa = __shfl_sync(0xffffffffu, a, from);
      const double ob = __shfl_sync(0xffffffffu, b, from);
      gb = fmax(fmax(gb, ob), fmin(ga, oa));
      ga = fmax(ga, oa);
    }
    double value = sums && gb > -CUDART_INF ? ga + gb : ga;
    if (g >= p.num_groups) value = -CUDART_INF;
    int place = 0;
#pragma unroll 1
    for (int o = 0; o < p.num_groups; ++o) {
      const double ov = __shfl_sync(0xffffffffu, value, o * lpg);
      place += ov > value || (ov == value && o < g);
    }
    const unsigned lanes =
        __ballot_sync(0xffffffffu, value > -CUDART_INF && place < p.topk_groups);
    open = 0;
#pragma unroll 1
    for (int o = 0; o < p.num_groups; ++o) open |= ((lanes >> (o * lpg)) & 1u) << o;
  }
  // keys as ordered integers, 0: not to be picked
  uint64_t* order = reinterpret_cast<uint64_t*>(key);
#pragma unroll 1
  for (int e = lane; e < p.E; e += 32) {
    double k = key[e];
    const bool out = !(k > -CUDART_INF) || !((open >> (p.num_groups > 1 ? e / per : 0)) & 1u);
    if (!p.bias && sums) k = static_cast<double>(logit_of(l, e));
    order[e] = out ? 0 : order_key64(k);
  }
  __syncwarp();
  mine = 0.f;
  mine_id = p.E;
  uint64_t best = 0;
  int id = 0;
  bool stale = true;  // this lane's best key was picked (or none is known yet)
#pragma unroll 1
  for (int j = 0; j < p.k; ++j) {
    if (stale) {
      best = 0;
#pragma unroll 1
      for (int e = lane; e < p.E; e += 32)
        if (order[e] > best) {
          best = order[e];
          id = e;
        }
    }
    __syncwarp();
    const uint32_t hi = __reduce_max_sync(0xffffffffu, static_cast<uint32_t>(best >> 32));
    if (hi == 0) break;
    const bool top = static_cast<uint32_t>(best >> 32) == hi;
    const uint32_t lo = __reduce_max_sync(0xffffffffu, top ? static_cast<uint32_t>(best) : 0u);
    const unsigned pick = __reduce_min_sync(
        0xffffffffu, top && static_cast<uint32_t>(best) == lo ? static_cast<unsigned>(id)
                                                              : 0xffffffffu);
    if (lane == j) mine_id = static_cast<int>(pick);
    stale = static_cast<int>(pick) % 32 == lane;
    if (stale) order[pick] = 0;
  }
  if (mine_id < p.E)
    mine = static_cast<float>(score64(logit_of(l, mine_id), m, total, p.scoring));
}

// Scores below this, in a row whose picks' sum is below 1/2, send its renormalised weights to 64
// bits: a sigmoid's exponential passes the largest f32 at a logit of -88.7 and a softmax score its
// last subnormal 103 below the row's maximum, but a share of the sum does not depend on how small
// its terms are.  (Next to a larger sum what is lost is under 2^-126, below any normal weight.)
constexpr float kTinyScore = 0x1p-100f, kSmallSum = 0.5f;

// The row's renormalised weights again, in 64 bits, from the ids its slots hold; by one warp.
// 1 / (1 + e^-l) and e^(l - m) as in route_row64: what is 0 in 64 bits counts as 0.
template <typename T>
__device__ __noinline__ void renormalise_row64(const RouteExpertsParams& p, int64_t row) {
  const int lane = threadIdx.x & 31;
  const T* l = static_cast<const T*>(p.logits) + row * p.stride;
  float m = -CUDART_INF_F;
  if (p.scoring == 0) {
#pragma unroll 1
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit_of(l, e));
    m = warp_max(m);
  }
  const int id = lane < p.k ? p.indices[row * p.k + lane] : p.E;
  const double r = id < p.E ? score64(logit_of(l, id), m, 1.0, p.scoring) : 0.0;
  const double sum = warp_sum(r);
  if (lane < p.k)
    p.weights[row * p.k + lane] =
        sum > 0.0 ? static_cast<float>(r / sum * static_cast<double>(p.scaling)) : 0.f;
}

// Writes the row's k slots from the pick that each lane holds (slot `lane`).
template <typename T>
__device__ __forceinline__ void store_row(const RouteExpertsParams& p, int64_t row, float r,
                                          int id) {
  const int lane = threadIdx.x & 31;
  bool tiny = false;
  if (p.renormalize) {
    const float sum = warp_sum(r);
    tiny = sum < kSmallSum && id < p.E && r < kTinyScore;
    r = sum > 0.f ? r / sum : r;
  }
  if (lane < p.k) {
    p.weights[row * p.k + lane] = r * p.scaling;
    p.indices[row * p.k + lane] = id;
  }
  if (__any_sync(0xffffffffu, tiny)) {
    __syncwarp();
    renormalise_row64<T>(p, row);
  }
}

// Every row in 64 bits: groups so uneven to the lanes that one would hold more than the 16 experts
// the kernel below keeps in registers.  16384 rows of 510 experts in 5 groups: 141 us.
template <typename T>
__global__ void __launch_bounds__(kWarps * 32)
    route_experts64_kernel(const __grid_constant__ RouteExpertsParams p) {
  extern __shared__ double smem_d[];
  const int warp = threadIdx.x >> 5;
  double* key = smem_d + warp * row64_scratch(p.E);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kWarps + warp; row < p.num_tokens;
       row += static_cast<int64_t>(gridDim.x) * kWarps) {
    float r;
    int id;
    route_row64<T>(p, row, key, r, id);
    store_row<T>(p, row, r, id);
    __syncwarp();
  }
}

__device__ __forceinline__ float redux_max(float v) {
  float r;
  asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
  return r;
}

// One row per warp, 32-bit keys in registers.  Lane l holds `bs` <= VPT consecutive experts (of one
// group: lpg = 32 / num_groups lanes per group), so lane order is expert order.
//
// Picks: the k-th largest of the 32 lane maxima (k rounds of a warp maximum) is a lower bound of
// the k-th largest key, so the keys at or above it -- a few more than k -- are the only
// candidates; they are compacted into shared memory in expert order, one per lane (two with
// more than 32), and each counts the candidates before it: that count is its slot.  No round
// depends on the one before, as k warp argmax rounds would.
//
// Keys that are logits are exact.  With a bias the key s + b is off by at most `delta`; two
// candidates nearer than 2 delta that are not the same numbers, or two groups nearer than their
// sums' error, send the row to route_row64, which decides in 64 bits (one row in thousands).
//
// delta, here and in the kernel below, with h = 2^-24 and CUDA's stated bounds (expf 2 ulp, __expf
// 2 + 1.173 |x| ulp, __fdividef 2 ulp, an ulp being at most 2 h):
//   sigmoid 1 / (1 + e), e = exp(-x): the relative error of e, at most (4 + 2.35 |x|) h, counts
//     s (1 - s) times, h for 1 + e and 4 h for the quotient s times.  s (1 - s) (4 + 2.35 |x|) + 5 s
//     is below 5.6 for every x: under 3.4e-7 of the 4e-7 taken.
//   softmax exp(-d) / S, d = m - x: a key's own part is d h for the difference, (4 + 2.35 d) h for
//     the exponential and h for the product, exp(-d) (5 + 3.35 d) <= 5 times h / S.  What all keys
//     of a row share is the error of 1 / S: the terms' (d + 4) h weighted by exp(-d) / S, where the
//     mean of d is at most ln 512 = 6.3 (it is the entropy less ln S), up to 36 additions of a
//     term (32 in a lane, 4 across) and the division, under 48 h.  Together 53 h / S = 3.2e-6 of
//     the largest score 1 / S; 6e-6 is taken.
//   the sum s + b: one rounding, h |s + b|; 1.2e-7 of the largest candidate is twice that.
// The bound t lies 4 delta below the k-th block maximum: a true pick is above the k-th true key,
// so its computed key is at most 2 delta below the k-th computed one.  A group's sum of two keys
// is off by 2 delta and four roundings, so two groups by 4 delta + 8 h of the larger key.
//
// Measured, 16384 rows, eight sets of inputs in turn: 512 experts top 10 17.2 us, 256 top 16 18.4
// us (0.9 TB/s), with sigmoid scores and a bias 39 us, 60 experts in 5 groups top 8 17 us.
template <typename T, int VPT, bool kBias, bool kGroups>
__global__ void __launch_bounds__(kFastWarps * 32)
    route_experts_kernel(const __grid_constant__ RouteExpertsParams p, int bs, int lpg, int vec) {
  extern __shared__ double smem_d[];
  __shared__ alignas(16) float s_key[kFastWarps][kMaxCand];
  __shared__ uint16_t s_id[kFastWarps][kMaxCand];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const float kNone = -CUDART_INF_F;
  float* ck = s_key[warp];
  uint16_t* cid = s_id[warp];
  const int per = p.E / p.num_groups;
  // this lane's experts: [e0, e0 + n)
  const int g = kGroups ? lane / lpg : 0;
  int e0 = kGroups ? g * per + (lane % lpg) * bs : lane * bs;
  int n = min(bs, (kGroups ? (g + 1) * per : p.E) - e0);
  if (kGroups && g >= p.num_groups) n = 0;
  n = max(n, 0);
  if (n == 0) e0 = 0;
  float b[kBias ? VPT : 1];
  if (kBias) {
#pragma unroll
    for (int i = 0; i < VPT; ++i) b[i] = i < n ? __ldg(p.bias + e0 + i) : 0.f;
  }
  const bool sums = kGroups && p.group_score != 0;
  const bool need_total = p.scoring == 0 && (kBias || sums || !p.renormalize);
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kFastWarps + warp; row < p.num_tokens;
       row += static_cast<int64_t>(gridDim.x) * kFastWarps) {
    const T* l = static_cast<const T*>(p.logits) + row * p.stride;
    float v[VPT];
    if (vec) {  // n is 0 or bs, and bs a multiple of 16 bytes
      constexpr int kPer = 16 / sizeof(T);
#pragma unroll
      for (int c = 0; c < (VPT + kPer - 1) / kPer; ++c) {
        alignas(16) T q[kPer];
        if (c * kPer < n)
          *reinterpret_cast<uint4*>(q) = __ldg(reinterpret_cast<const uint4*>(l + e0) + c);
#pragma unroll
        for (int i = 0; i < kPer; ++i)
          if (c * kPer + i < VPT) v[c * kPer + i] = c * kPer < n ? Elem<T>::to_f(q[i]) : kNone;
      }
    } else {
#pragma unroll
      for (int i = 0; i < VPT; ++i) v[i] = i < n ? Elem<T>::to_f(l[e0 + i]) : kNone;
    }
    float m = kNone;
#pragma unroll
    for (int i = 0; i < VPT; ++i) {
      v[i] = v[i] == v[i] ? v[i] : kNone;
      m = fmaxf(m, v[i]);
    }
    const float lane_max = m;
    float total = 1.f, delta = 0.f;
    if (p.scoring == 0) {
      m = redux_max(m);
      if (need_total) {
        total = 0.f;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          if (v[i] > kNone) total += expf(v[i] - m);
        total = warp_sum(total);
      }
    }
    const float inv = 1.f / total;
    auto score = [&](float x) -> float {
      return p.scoring == 0 ? expf(x - m) * inv : 1.f / (1.f + expf(-x));
    };
    bool unsure = false;
    float top = lane_max;
    float group_value = kNone, magnitude = 0.f;
    if (kBias || sums) {
      float a = kNone, a2 = kNone;
#pragma unroll
      for (int i = 0; i < VPT; ++i) {
        float x = kNone;
        if (v[i] > kNone) {
          x = score(v[i]) + (kBias ? b[i] : 0.f);
          x = x == x ? x : kNone;
        }
        if (kBias) v[i] = x;
        a2 = fmaxf(a2, fminf(a, x));
        a = fmaxf(a, x);
      }
      if (kBias) top = a;
      // score(m) = 1 / total is the largest softmax score
      delta = p.scoring == 0 ? 6e-6f * inv : 4e-7f;
      if (sums) {
        group_value = a;
        float second = a2;
        for (int o = 1; o < lpg; ++o) {  // the other lanes of the group, in turn
          const int from = g * lpg + (lane - g * lpg + o) % lpg;
          const float oa = __shfl_sync(0xffffffffu, a, from & 31);
          const float o2 = __shfl_sync(0xffffffffu, a2, from & 31);
          second = fmaxf(fmaxf(second, o2), fminf(group_value, oa));
          group_value = fmaxf(group_value, oa);
        }
        if (group_value > kNone) magnitude = fabsf(group_value);
        if (second > kNone) {
          magnitude = fmaxf(magnitude, fabsf(second));
          group_value += second;
        }
      }
    }
    if (kGroups) {
      if (!sums) {
        group_value = top;
        for (int o = 1; o < lpg; ++o)
          group_value = fmaxf(group_value, __shfl_sync(0xffffffffu, top,
                                                       (g * lpg + (lane - g * lpg + o) % lpg) & 31));
        magnitude = fabsf(group_value);
      }
      if (g >= p.num_groups) group_value = kNone;
      // a group's place among the groups, and whether the 32-bit values may mislead about it
      const bool exact = !kBias && !sums;
      const float slack = exact ? -1.f : 4.f * delta + 5e-7f * magnitude;
      int place = 0;
      for (int o = 0; o < p.num_groups; ++o) {
        const float ov = __shfl_sync(0xffffffffu, group_value, o * lpg);
        place += ov > group_value || (ov == group_value && o < g);
        unsure |= o != g && fabsf(ov - group_value) <= slack;
      }
      unsure = unsure && group_value > kNone;
      if (!(place < p.topk_groups)) {
#pragma unroll
        for (int i = 0; i < VPT; ++i) v[i] = kNone;
        top = kNone;
      }
    }
    // lower bound of the k-th largest key
    float t = kNone, cur = top, best = kNone;
    for (int j = 0; j < p.k; ++j) {
      t = redux_max(cur);
      if (j == 0) best = t;
      if (!(t > kNone)) break;
      cur = cur == t ? kNone : cur;
    }
    if (kBias) {
      delta += 1.2e-7f * fmaxf(fabsf(best), t > kNone ? fabsf(t) : 0.f);
      t -= 4.f * delta;
      if (best == CUDART_INF_F) {  // a bias of +inf: no candidates here, all in 64 bits
        unsure = true;
        t = CUDART_NAN_F;
      }
    }
    int mine = 0;
#pragma unroll
    for (int i = 0; i < VPT; ++i) mine += v[i] >= t && v[i] > kNone;
    int before = mine;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, o);
      if (lane >= o) before += up;
    }
    const int count = __shfl_sync(0xffffffffu, before, 31);
    before -= mine;
    float r = 0.f;
    int id = p.E;
    if (count <= kMaxCand) {
      ck[lane] = kNone;
      ck[lane + 32] = kNone;
      __syncwarp();
#pragma unroll
      for (int i = 0; i < VPT; ++i)
        if (v[i] >= t && v[i] > kNone) {
          ck[before] = v[i];
          cid[before] = static_cast<uint16_t>(e0 + i);
          ++before;
        }
      __syncwarp();
      int place[2] = {0, 0};
      const float key[2] = {ck[lane], ck[lane + 32]};
      const int halves = count > 32 ? 2 : 1;
      for (int i = 0; i < count; i += 4) {
        const float4 o4 = *reinterpret_cast<const float4*>(ck + i);
        const float o[4] = {o4.x, o4.y, o4.z, o4.w};
#pragma unroll
        for (int q = 0; q < 4; ++q) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            if (h == halves) break;
            const int at = lane + 32 * h;
            place[h] += o[q] > key[h] || (o[q] == key[h] && i + q < at);
            if (kBias && i + q != at && at < count && fabsf(o[q] - key[h]) <= 2.f * delta) {
              // the same numbers tie for certain
              const int x = cid[i + q], y = cid[at];
              unsure |= Elem<T>::to_f(l[x]) != Elem<T>::to_f(l[y]) || p.bias[x] != p.bias[y];
            }
          }
        }
      }
      __syncwarp();
      // slot `place` takes this candidate: through shared memory to the lane of that slot
      const int ids[2] = {lane < count ? cid[lane] : 0, lane + 32 < count ? cid[lane + 32] : 0};
      __syncwarp();
#pragma unroll
      for (int h = 0; h < 2; ++h)
        if (lane + 32 * h < count && place[h] < p.k) cid[place[h]] = static_cast<uint16_t>(ids[h]);
      __syncwarp();
      if (lane < p.k && lane < count) {
        id = cid[lane];
        r = score(logit_of(l, id));
      }
    } else if (kBias) {
      unsure = true;
    } else {
      // many equal keys: k warp argmax rounds
      for (int j = 0; j < p.k; ++j) {
        float x = kNone;
        int at = 0;
#pragma unroll
        for (int i = 0; i < VPT; ++i)
          if (v[i] > x) {
            x = v[i];
            at = i;
          }
        const float w = redux_max(x);
        const int first = __ffs(__ballot_sync(0xffffffffu, x == w)) - 1;
        const int pick = __shfl_sync(0xffffffffu, e0 + at, first);
        if (lane == first) {
#pragma unroll
          for (int i = 0; i < VPT; ++i)
            if (i == at) v[i] = kNone;
        }
        if (lane == j) {
          id = pick;
          r = score(logit_of(l, id));
        }
      }
    }
    if ((kBias || sums) && __any_sync(0xffffffffu, unsure))
      route_row64<T>(p, row, smem_d + warp * row64_scratch(p.E), r, id);
    store_row<T>(p, row, r, id);
    __syncwarp();
  }
}

// ---- several rows per warp, k <= 8 -------------------------------------------------------------

__device__ __forceinline__ void order2(float& a, float& b) {  // a >= b
  const float hi = fmaxf(a, b);
  b = fminf(a, b);
  a = hi;
}

// Descending sort of 8 (19 comparators) and of a bitonic sequence of 8.
__device__ __forceinline__ void sort8(float (&x)[8]) {
  order2(x[0], x[1]); order2(x[2], x[3]); order2(x[4], x[5]); order2(x[6], x[7]);
  order2(x[0], x[2]); order2(x[1], x[3]); order2(x[4], x[6]); order2(x[5], x[7]);
  order2(x[1], x[2]); order2(x[5], x[6]);
  order2(x[0], x[4]); order2(x[1], x[5]); order2(x[2], x[6]); order2(x[3], x[7]);
  order2(x[2], x[4]); order2(x[3], x[5]);
  order2(x[1], x[2]); order2(x[3], x[4]); order2(x[5], x[6]);
}
__device__ __forceinline__ void sort_bitonic8(float (&x)[8]) {
#pragma unroll
  for (int d = 4; d > 0; d >>= 1)
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if ((i & d) == 0) order2(x[i], x[i + d]);
}

constexpr int kRowCand = 16;  // candidates of a row

// The float of a candidate's order-preserving key.
__device__ __forceinline__ float from_key(uint64_t c) {
  const uint32_t k = static_cast<uint32_t>(c >> 32);
  return __uint_as_float((k >> 31) ? k & 0x7fffffffu : ~k);
}

// Ranks the `count` candidates (key << 32 | ~id) of each of a warp's rows by sigmoid + bias in 64
// bits, ties to the lower id; cand is overwritten.
template <typename T, int LPR>
__device__ __noinline__ void rank64(const T* l, const float* __restrict__ bias, uint64_t* cand,
                                    uint64_t* ranked, int count) {
  const int q = (threadIdx.x & 31) % LPR;
#pragma unroll 1
  for (int i = q; i < count; i += LPR) {
    const uint64_t c = cand[i];
    const int id = static_cast<int>(~static_cast<uint32_t>(c));
    ranked[i] = c;  // by position; its key in 64 bits in cand
    cand[i] = order_key64(score64(Elem<T>::to_f(l[id]), 0.f, 1.0, 1) +
                          static_cast<double>(bias[id]));
  }
  __syncwarp();
  uint64_t mine[kRowCand / LPR];
  int at[kRowCand / LPR];
#pragma unroll
  for (int h = 0; h < kRowCand / LPR; ++h) {
    const int i = q + h * LPR;
    at[h] = 0;
    mine[h] = 0;
    if (i < count) {
      mine[h] = ranked[i];
      const uint64_t key = cand[i];
#pragma unroll 1
      for (int j = 0; j < count; ++j)  // ~id: larger for the lower id
        at[h] += cand[j] > key || (cand[j] == key && static_cast<uint32_t>(ranked[j]) >
                                                         static_cast<uint32_t>(mine[h]));
    }
  }
  __syncwarp();
#pragma unroll
  for (int h = 0; h < kRowCand / LPR; ++h)
    if (mine[h]) ranked[at[h]] = mine[h];
  __syncwarp();
}
constexpr int kRowWarps = 4;

// LPR lanes per row, each with up to VPL experts in registers; k <= 8.
//
// As in the kernel above the picks come from a lower bound t of the k-th largest key and a
// ranking of the keys at or above it, with less work per row: t is the k-th largest of the
// maxima of small blocks (VPL / 8 experts of a lane), sorted by a network in each lane and merged
// over the row's lanes.  With 32 blocks and k = 8 about ten keys reach t.  The work is
// instructions, not bytes: a whole warp per row spent 560 warp instructions on a row of 128
// experts.
//
// Expert i of a lane is base + (i / 4) * cs + i % 4: without groups the row's lanes take pieces of
// four in turn (64 contiguous bytes of f32), with groups a lane holds one stretch of one group.
// NaN needs no care where it is compared: it is never >= t nor > -inf.
//
// Measured, eight sets of inputs in turn: 65536 x 128 f32 in 16.6 us (2.3 TB/s; 0.66 of the issue
// slots busy, 176 instructions a row), 16384 x 256 with sigmoid scores 10.2 us, with a bias 13.5
// us, with 8 groups as well 21.3 us (the 64-bit check of a close pair of groups, one row in 20000,
// is 4 us of it).  Rows with more than 16 keys at the bound go to route_row64 too, one after the
// other: 65536 x 128 with every other row constant takes 88 us.
template <typename T, int LPR, int VPL, bool kBias>
__global__ void __launch_bounds__(kRowWarps * 32, VPL <= 16 ? 8 : 6)
    route_experts_rows_kernel(const __grid_constant__ RouteExpertsParams p, int bs, int lpg,
                              int vec) {
  extern __shared__ double smem_d[];
  constexpr int RPW = 32 / LPR;
  // (order-preserving key, ~id) of the candidates; then key and id by place
  __shared__ alignas(16) uint64_t s_cand[kRowWarps][RPW][kRowCand];
  __shared__ uint64_t s_rank[kRowWarps][RPW][kRowCand];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, q = lane % LPR;
  const float kNone = -CUDART_INF_F;
  uint64_t* cand = s_cand[warp][sub];
  uint64_t* ranked = s_rank[warp][sub];
  const bool groups = p.num_groups > 1;
  const int per = p.E / p.num_groups;
  const int g = groups ? q / lpg : 0;
  const int cs = groups ? 4 : 4 * LPR;
  const int base = groups ? g * per + (q % lpg) * bs : 4 * q;
  const int lim = groups ? min(bs, per - (q % lpg) * bs) : p.E - base;
  const bool sums = groups && p.group_score != 0;
  const bool need_total = p.scoring == 0 && (kBias || sums || !p.renormalize);
  auto row_max = [&](float x) {
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, d));
    return x;
  };
  auto row_sum = [&](float x) {
#pragma unroll
    for (int d = LPR / 2; d > 0; d >>= 1) x += __shfl_xor_sync(0xffffffffu, x, d);
    return x;
  };
  for (int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kRowWarps + warp) * RPW;
       row0 < p.num_tokens; row0 += static_cast<int64_t>(gridDim.x) * kRowWarps * RPW) {
    const int64_t row = row0 + sub;
    const bool live = row < p.num_tokens;
    const T* l = static_cast<const T*>(p.logits) + (live ? row : row0) * p.stride;
    float v[VPL];
#pragma unroll
    for (int c = 0; c < VPL / 4; ++c) {
      if (vec) {  // every piece of four is whole and aligned
        struct alignas(4 * sizeof(T)) Four { T x[4]; };
        Four f;
        const bool in = c * cs < lim;
        if (in) f = *reinterpret_cast<const Four*>(l + base + c * cs);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[4 * c + i] = in ? Elem<T>::to_f(f.x[i]) : kNone;
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          v[4 * c + i] = c * cs + i < lim ? Elem<T>::to_f(l[base + c * cs + i]) : kNone;
      }
    }
    float m = 0.f, inv = 1.f, delta = 0.f;
    if (need_total) {
      m = kNone;
#pragma unroll
      for (int i = 0; i < VPL; ++i) m = fmaxf(m, v[i]);
      m = row_max(m);
      float total = 0.f;
#pragma unroll
      for (int i = 0; i < VPL; ++i)
        if (v[i] > kNone) total += expf(v[i] - m);
      inv = 1.f / row_sum(total);
    }
    bool unsure = false;
    float a = kNone, a2 = kNone;  // the lane's two largest score + bias
    if (kBias || sums) {
      // fast exponentials and quotients: their errors are inside delta (a sigmoid's exponential is
      // off by (2 + 1.16 |x|) ulp, times s (1 - s): under one ulp of 1)
#pragma unroll
      for (int c = 0; c < VPL / 4; ++c) {
        float b[4] = {0.f, 0.f, 0.f, 0.f};
        if (kBias) {
          if (vec) {
            if (c * cs < lim) {
              const float4 b4 = __ldg(reinterpret_cast<const float4*>(p.bias + base + c * cs));
              b[0] = b4.x;
              b[1] = b4.y;
              b[2] = b4.z;
              b[3] = b4.w;
            }
          } else {
#pragma unroll
            for (int i = 0; i < 4; ++i)
              if (c * cs + i < lim) b[i] = __ldg(p.bias + base + c * cs + i);
          }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float at = v[4 * c + i];
          float x = p.scoring == 0 ? __expf(at - m) * inv : __fdividef(1.f, 1.f + __expf(-at));
          x = at > kNone ? x + b[i] : kNone;
          if (kBias) v[4 * c + i] = x;
          if (sums) {
            a2 = fmaxf(a2, fminf(a, x == x ? x : kNone));
            a = fmaxf(a, x);
          }
        }
      }
      // score(m) = inv is the largest softmax score
      delta = p.scoring == 0 ? 6e-6f * inv : 4e-7f;
    }
    // maxima of blocks
    float top[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      constexpr int kBlock = VPL >= 8 ? VPL / 8 : 1;
      top[j] = kNone;
#pragma unroll
      for (int i = 0; i < kBlock; ++i)
        if (j * kBlock + i < VPL) top[j] = fmaxf(top[j], v[(j * kBlock + i) % VPL]);
    }
    sort8(top);
    if (groups) {
      float value, magnitude;
      if (sums) {
        for (int d = 1; d < lpg; d <<= 1) {
          const float oa = __shfl_xor_sync(0xffffffffu, a, d);
          const float o2 = __shfl_xor_sync(0xffffffffu, a2, d);
          a2 = fmaxf(fmaxf(a2, o2), fminf(a, oa));
          a = fmaxf(a, oa);
        }
        value = a2 > kNone ? a + a2 : a;
        magnitude = fmaxf(fabsf(a), a2 > kNone ? fabsf(a2) : 0.f);
      } else {
        value = top[0];
        for (int d = 1; d < lpg; d <<= 1)
          value = fmaxf(value, __shfl_xor_sync(0xffffffffu, value, d));
        magnitude = fabsf(value);
      }
      // a group's place among the groups, and whether the 32-bit values may mislead about it
      const float slack = !kBias && !sums ? -1.f : 4.f * delta + 5e-7f * magnitude;
      int place = 0;
      for (int o = 0; o < p.num_groups; ++o) {
        const float ov = __shfl_sync(0xffffffffu, value, o * lpg, LPR);
        place += ov > value || (ov == value && o < g);
      }
      const bool chosen = place < p.topk_groups;
      // the best group left out, and whether a chosen one is nearer to it than the errors
      const float out = row_max(chosen ? kNone : value);
      const float reach = row_max(chosen ? kNone : slack);
      unsure = chosen && value > kNone && out > kNone && value - out <= fmaxf(slack, reach);
      if (!chosen) {
#pragma unroll
        for (int i = 0; i < VPL; ++i) v[i] = kNone;
#pragma unroll
        for (int j = 0; j < 8; ++j) top[j] = kNone;
      }
    }
    // lower bound of the k-th largest key
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) {
      float other[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) other[j] = __shfl_xor_sync(0xffffffffu, top[j], d);
#pragma unroll
      for (int j = 0; j < 8; ++j) top[j] = fmaxf(top[j], other[7 - j]);
      sort_bitonic8(top);
    }
    float t = top[0];
#pragma unroll
    for (int j = 1; j < 8; ++j) t = j < p.k ? top[j] : t;
    if (kBias) {
      delta += 1.2e-7f * fmaxf(fabsf(top[0]), t > kNone ? fabsf(t) : 0.f);
      t -= 4.f * delta;
    }
    t = fmaxf(t, -3.402823466e38f);  // an unavailable expert is no candidate
    // renormalised softmax weights need no common factor
    if (p.scoring == 0 && !need_total) m = top[0];
    // candidates, into the row's list
    uint32_t mask = 0;
#pragma unroll
    for (int i = 0; i < VPL; ++i)
      if (v[i] >= t) mask |= 1u << i;
    const int mine = __popc(mask);
    int before = mine;
#pragma unroll
    for (int d = 1; d < LPR; d <<= 1) {
      const int up = __shfl_up_sync(0xffffffffu, before, d, LPR);
      if (q >= d) before += up;
    }
    const int count = __shfl_sync(0xffffffffu, before, LPR - 1, LPR);
    before -= mine;
#pragma unroll
    for (int i = q; i < kRowCand; i += LPR) cand[i] = 0;
    __syncwarp();
    const bool fits = count <= kRowCand;
    if (!fits) mask = 0;
    unsure |= !fits;
    while (mask) {
      const int i = __ffs(mask) - 1;
      mask &= mask - 1;
      const int id = base + (i >> 2) * cs + (i & 3);
      float x = Elem<T>::to_f(l[id]);
      if (kBias) {
        x = p.scoring == 0 ? __expf(x - m) * inv : __fdividef(1.f, 1.f + __expf(-x));
        x += __ldg(p.bias + id);
      }
      const uint32_t b = __float_as_uint(x + 0.f);  // -0 as +0
      const uint32_t key = (b >> 31) ? ~b : (b | 0x80000000u);
      cand[before] = (static_cast<uint64_t>(key) << 32) | static_cast<uint32_t>(~id);
      ++before;
    }
    __syncwarp();
    // each lane ranks every LPR-th candidate: larger key first, then the lower id
    const int most = min(__reduce_max_sync(0xffffffffu, count), kRowCand);
#pragma unroll
    for (int h = 0; h < kRowCand / LPR; ++h) {
      if (h * LPR < most) {
        const uint64_t x = cand[q + h * LPR];
        int at = 0;
        for (int j = 0; j < most; j += 2) {
          const ulonglong2 o = *reinterpret_cast<const ulonglong2*>(cand + j);
          at += o.x > x;
          at += o.y > x;
        }
        if (x) ranked[at] = x;
      }
    }
    __syncwarp();
    if (kBias) {
      // is every pick certainly ahead of the next candidate?
      bool close = false;
      for (int j = q; j < min(p.k, count - 1) && fits; j += LPR)
        close |= from_key(ranked[j]) - from_key(ranked[j + 1]) <= 2.f * delta;
      if (__any_sync(0xffffffffu, close)) {
        if (p.scoring == 0) {
          unsure |= close;
        } else {  // rank again in 64 bits; every candidate that matters is in the list
          rank64<T, LPR>(l, p.bias, cand, ranked, fits ? count : 0);
        }
      }
    }
    // each lane takes every LPR-th slot
    constexpr int kSlots = (8 + LPR - 1) / LPR;
    const int picks = fits ? min(count, p.k) : 0;
    float r[kSlots], sum = 0.f;
    int id[kSlots];
#pragma unroll
    for (int h = 0; h < kSlots; ++h) {
      const int j = q + h * LPR;
      r[h] = 0.f;
      id[h] = p.E;
      if (j < picks) {
        const uint64_t c = ranked[j];
        id[h] = static_cast<int>(~static_cast<uint32_t>(c));
        const float x = Elem<T>::to_f(l[id[h]]);
        r[h] = p.scoring == 0 ? expf(x - m) * inv : 1.f / (1.f + expf(-x));
        sum += r[h];
      }
    }
    float scale = p.scaling;
    bool tiny = false;
    if (p.renormalize) {
      sum = row_sum(sum);
      scale = sum > 0.f ? p.scaling / sum : scale;
      if (sum < kSmallSum) {
        tiny = isinf(scale);
#pragma unroll
        for (int h = 0; h < kSlots; ++h) tiny |= id[h] < p.E && r[h] < kTinyScore;
      }
    }
    if (live) {
#pragma unroll
      for (int h = 0; h < kSlots; ++h)
        if (q + h * LPR < p.k) {
          p.weights[row * p.k + q + h * LPR] = r[h] * scale;
          p.indices[row * p.k + q + h * LPR] = id[h];
        }
    }
    // rows of tiny scores, one after the other (those of the next loop are stored again there)
    unsigned left = __ballot_sync(0xffffffffu, tiny && live);
    if (left) __syncwarp();  // reads the ids stored above
    while (left) {
      const int s = (__ffs(left) - 1) / LPR;
      left &= ~(((1u << LPR) - 1u) << (s * LPR));
      renormalise_row64<T>(p, row0 + s);
      __syncwarp();
    }
    // rows that 32 bits do not decide, or with many equal keys, one after the other
    left = __ballot_sync(0xffffffffu, unsure && live);
    while (left) {
      const int s = (__ffs(left) - 1) / LPR;
      left &= ~(((1u << LPR) - 1u) << (s * LPR));
      float r1;
      int id1;
      route_row64<T>(p, row0 + s, smem_d + warp * row64_scratch(p.E), r1, id1);
      store_row<T>(p, row0 + s, r1, id1);
      __syncwarp();
    }
    __syncwarp();
  }
}

// ---- gradient ----------------------------------------------------------------------------------

__device__ __forceinline__ void bulk_store(void* dst, const void* src, uint32_t bytes) {
  asm volatile("cp.async.bulk.global.shared::cta.bulk_group [%0], [%1], %2;" ::"l"(dst),
               "r"(smem_addr(src)), "r"(bytes)
               : "memory");
  asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void bulk_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(N) : "memory");
}

// Gradients that are zero except at the picks:
//     softmax, renormalised:  dl_j = w_j (g_j - G),            G = sum_i g_i w_i / c
//     sigmoid:                dl_j = w_j (g_j - G) (1 - s_j),  G = 0 unless renormalised
// so at most the picks' logits are read.  LPR lanes per row, a lane per slot (k <= LPR): a warp
// reads the slots of 32 / LPR rows at once, drops their gradients into a tile of zeros in shared
// memory and sends the tile out in one bulk copy; two tiles in turn, and the places written
// are cleared once the copy has read them.  65536 x 128 f32 in 8.3 us, 4.8 TB/s of slots read and
// gradients written; held by shared memory, the match over the warp and the shuffles (short
// scoreboard and MIO stalls), not yet by the bytes (a warp per row, with its own stores, took 162
// instructions a row and 33 us).
template <typename T, int LPR>
__global__ void __launch_bounds__(kRowWarps * 32)
    route_experts_backward_kernel(RouteExpertsBackwardParams p, int bulk) {
  extern __shared__ __align__(128) char smem_c[];
  constexpr int RW = 32 / LPR;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int sub = lane / LPR, q = lane % LPR;
  const int tile = RW * p.E;                              // elements
  const int pitch = (tile * static_cast<int>(sizeof(T)) + 15) & ~15;  // bytes
  char* base = smem_c + warp * 2 * pitch;
  const int64_t stride = static_cast<int64_t>(gridDim.x) * kRowWarps * RW;
  int64_t row0 = (static_cast<int64_t>(blockIdx.x) * kRowWarps + warp) * RW;
  // the next rows' picks are loaded while these rows are written
  float gn = 0.f, wn = 0.f;
  int idn = -1;
  auto load = [&](int64_t r0) {
    const int64_t r = r0 + sub;
    idn = -1;
    if (q < p.k && r < p.num_tokens) {
      gn = __ldcs(p.grad_weights + r * p.k + q);
      wn = __ldcs(p.weights + r * p.k + q);
      idn = __ldcs(p.indices + r * p.k + q);
    }
  };
  float xn = 0.f;
  auto load_logit = [&](int64_t r0) {
    if (p.scoring != 0 && idn >= 0 && idn < p.E)
      xn = logit_of(static_cast<const T*>(p.logits) + (r0 + sub) * p.stride, idn);
  };
  load(row0);
  const int tiles = row0 + stride < p.num_tokens ? 2 : 1;
  for (int i = lane * 16; i < tiles * pitch; i += 512)
    *reinterpret_cast<uint4*>(base + i) = make_uint4(0, 0, 0, 0);
  load_logit(row0);
  int held[2] = {-1, -1};  // place this lane wrote in each tile
  int side = 0;
  for (; row0 < p.num_tokens; row0 += stride) {
    const bool ok = idn >= 0 && idn < p.E;
    const int id = ok ? idn : 0;
    const float g = ok ? gn : 0.f, w = ok ? wn : 0.f;
    const float x = xn;
    load(row0 + stride);
    float d = g * w;
    if (p.renormalize) {
      float G = d;
#pragma unroll
      for (int o = LPR / 2; o > 0; o >>= 1) G += __shfl_xor_sync(0xffffffffu, G, o);
      d = w * (g - G / p.scaling);
    }
    if (p.scoring != 0) d *= 1.f / (1.f + expf(x));
    T* buf = reinterpret_cast<T*>(base + side * pitch);
    bulk_wait_read<1>();  // the copy before the last, out of this tile, has read it
    __syncwarp();
    if (held[side] >= 0) buf[held[side]] = Elem<T>::from_f(0.f);
    __syncwarp();
    const int at = ok ? sub * p.E + id : -1;
    // one id twice in a row: the first lane of it adds the others' in slot order
    const unsigned peers = __match_any_sync(0xffffffffu, ok ? at : -1 - lane);
    const bool first = (peers & ((1u << lane) - 1u)) == 0;
    if (__any_sync(0xffffffffu, ok && !first)) {
      float sum = 0.f;
      for (int j = 0; j < 32; ++j) {
        const float o = __shfl_sync(0xffffffffu, d, j);
        if ((peers >> j) & 1u) sum += o;
      }
      d = sum;
    }
    if (ok && first) buf[at] = Elem<T>::from_f(d);
    held[side] = ok && first ? at : -1;
    const int rows = static_cast<int>(min(static_cast<int64_t>(RW), p.num_tokens - row0));
    T* out = static_cast<T*>(p.grad_logits) + row0 * p.E;
    const uint32_t bytes = rows * p.E * sizeof(T);
    if (bulk && bytes % 16 == 0) {
      asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
      __syncwarp();
      if (lane == 0) bulk_store(out, buf, bytes);
    } else {
      __syncwarp();
      for (int i = lane; i < rows * p.E; i += 32) out[i] = buf[i];
      asm volatile("cp.async.bulk.commit_group;" ::: "memory");
    }
    __syncwarp();
    side ^= 1;
    load_logit(row0 + stride);
  }
  bulk_wait_read<0>();
}

// Softmax weights that are not renormalised: every expert has a gradient,
//     dl_e = s_e (c g_e - sum_i g_i w_i)
// One row per warp, the picks' share through a row of zeros in shared memory.
template <typename T>
__global__ void __launch_bounds__(kFastWarps * 32)
    route_experts_backward_dense_kernel(RouteExpertsBackwardParams p) {
  extern __shared__ float smem_f[];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  float* ds = smem_f + warp * p.E;
  for (int e = lane; e < p.E; e += 32) ds[e] = 0.f;
  __syncwarp();
  for (int64_t row = static_cast<int64_t>(blockIdx.x) * kFastWarps + warp; row < p.num_tokens;
       row += static_cast<int64_t>(gridDim.x) * kFastWarps) {
    const T* l = static_cast<const T*>(p.logits) + row * p.stride;
    T* out = static_cast<T*>(p.grad_logits) + row * p.E;
    float g = 0.f, w = 0.f;
    int id = -1;
    if (lane < p.k) {
      id = p.indices[row * p.k + lane];
      if (id >= 0 && id < p.E) {
        g = p.grad_weights[row * p.k + lane];
        w = p.weights[row * p.k + lane];
      } else {
        id = -1;
      }
    }
    float m = -CUDART_INF_F, total = 0.f;
    for (int e = lane; e < p.E; e += 32) m = fmaxf(m, logit_of(l, e));
    m = warp_max(m);
    for (int e = lane; e < p.E; e += 32) {
      const float x = logit_of(l, e);
      if (x > -CUDART_INF_F) total += expf(x - m);
    }
    const float inv = 1.f / warp_sum(total);
    const float D = warp_sum(g * w);
    // one id twice in a row adds up in slot order
    const unsigned peers = __match_any_sync(0xffffffffu, id >= 0 ? id : -1 - lane);
    if (!__any_sync(0xffffffffu, id >= 0 && (peers & (peers - 1)) != 0)) {
      if (id >= 0) ds[id] = g * p.scaling;
    } else {
      for (int j = 0; j < p.k; ++j) {
        if (lane == j && id >= 0) ds[id] += g * p.scaling;
        __syncwarp();
      }
    }
    __syncwarp();
    for (int e = lane; e < p.E; e += 32) {
      const float x = logit_of(l, e);
      out[e] = Elem<T>::from_f(x > -CUDART_INF_F ? expf(x - m) * inv * (ds[e] - D) : 0.f);
    }
    __syncwarp();
    if (id >= 0) ds[id] = 0.f;
    __syncwarp();
  }
}

int blocks_for(int64_t rows, int num_sms) {
  const int64_t b = (rows + kWarps - 1) / kWarps, cap = static_cast<int64_t>(num_sms) * 8;
  return static_cast<int>(b < cap ? b : cap);
}

}  // namespace

namespace {

template <typename T, int VPT>
void launch_fast(const RouteExpertsParams& p, int bs, int lpg, int vec, int num_sms,
                 cudaStream_t s) {
  const int64_t blocks = (p.num_tokens + kFastWarps - 1) / kFastWarps;
  const int64_t cap = static_cast<int64_t>(num_sms) * 8;  // 64 warps on an SM
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  const bool groups = p.num_groups > 1;
  const bool may64 = p.bias || (groups && p.group_score != 0);
  const size_t smem = may64 ? sizeof(double) * kFastWarps * row64_scratch(p.E) : 0;
  if (p.bias) {
    if (groups)
      route_experts_kernel<T, VPT, true, true><<<grid, kFastWarps * 32, smem, s>>>(p, bs, lpg, vec);
    else
      route_experts_kernel<T, VPT, true, false><<<grid, kFastWarps * 32, smem, s>>>(p, bs, lpg, vec);
  } else {
    if (groups)
      route_experts_kernel<T, VPT, false, true><<<grid, kFastWarps * 32, smem, s>>>(p, bs, lpg, vec);
    else
      route_experts_kernel<T, VPT, false, false><<<grid, kFastWarps * 32, smem, s>>>(p, bs, lpg, vec);
  }
}

template <typename T, int LPR, int VPL>
void launch_rows(const RouteExpertsParams& p, int bs, int lpg, int num_sms, cudaStream_t s) {
  constexpr int rows = kRowWarps * (32 / LPR);
  const int64_t blocks = (p.num_tokens + rows - 1) / rows, cap = static_cast<int64_t>(num_sms) * 16;
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  const size_t smem = sizeof(double) * kRowWarps * row64_scratch(p.E);
  const int per = p.E / p.num_groups;
  const int vec = (p.num_groups > 1 ? bs % 4 == 0 && per % bs == 0 : p.E % 4 == 0) &&
                  p.stride % 4 == 0 &&
                  (reinterpret_cast<uintptr_t>(p.logits) & (4 * sizeof(T) - 1)) == 0 &&
                  (reinterpret_cast<uintptr_t>(p.bias) & 15u) == 0;
  if (p.bias)
    route_experts_rows_kernel<T, LPR, VPL, true><<<grid, kRowWarps * 32, smem, s>>>(p, bs, lpg, vec);
  else
    route_experts_rows_kernel<T, LPR, VPL, false><<<grid, kRowWarps * 32, smem, s>>>(p, bs, lpg,
                                                                                       vec);
}

// Whether the kernel of LPR lanes per row and VPL experts per lane can take p.
template <typename T, int LPR, int VPL>
bool try_rows(const RouteExpertsParams& p, int num_sms, cudaStream_t s) {
  if (LPR % p.num_groups != 0) return false;
  const int lpg = LPR / p.num_groups, bs = (p.E / p.num_groups + lpg - 1) / lpg;
  if (p.num_groups == 1 ? p.E > VPL * LPR : bs > VPL) return false;
  launch_rows<T, LPR, VPL>(p, bs, lpg, num_sms, s);
  return true;
}

template <typename T>
void launch_route(const RouteExpertsParams& p, int num_sms, cudaStream_t s) {
  if (p.k <= 8) {
    if (p.num_groups == 1 && p.E <= 16) return launch_rows<T, 4, 4>(p, 4, 4, num_sms, s);
    if (try_rows<T, 4, 16>(p, num_sms, s) || try_rows<T, 8, 16>(p, num_sms, s) ||
        try_rows<T, 16, 16>(p, num_sms, s) || try_rows<T, 16, 32>(p, num_sms, s))
      return;
  }
  const int lpg = 32 / p.num_groups;
  const int per = p.E / p.num_groups;
  const int bs = (per + lpg - 1) / lpg;
  const int vec = (bs * sizeof(T)) % 16 == 0 && per % bs == 0 && (p.stride * sizeof(T)) % 16 == 0 &&
                  (reinterpret_cast<uintptr_t>(p.logits) & 15u) == 0;
  if (bs == 1) return launch_fast<T, 1>(p, bs, lpg, vec, num_sms, s);
  if (bs == 2) return launch_fast<T, 2>(p, bs, lpg, vec, num_sms, s);
  if (bs <= 4) return launch_fast<T, 4>(p, bs, lpg, vec, num_sms, s);
  if (bs <= 8) return launch_fast<T, 8>(p, bs, lpg, vec, num_sms, s);
  if (bs <= 16) return launch_fast<T, 16>(p, bs, lpg, vec, num_sms, s);
  // groups so uneven to the lanes that a lane would hold more than 16 experts
  const size_t smem = sizeof(double) * kWarps * row64_scratch(p.E);
  route_experts64_kernel<T><<<blocks_for(p.num_tokens, num_sms), kWarps * 32, smem, s>>>(p);
}

}  // namespace

int launch_route_experts(int dtype, const RouteExpertsParams& p, int num_sms, cudaStream_t s) {
  if (p.num_tokens <= 0) return 0;
  if (dtype == kF32) launch_route<float>(p, num_sms, s);
  else if (dtype == kBF16) launch_route<__nv_bfloat16>(p, num_sms, s);
  else launch_route<__half>(p, num_sms, s);
  return 0;
}

namespace {
template <typename T, int LPR>
void launch_backward_picks(const RouteExpertsBackwardParams& p, int num_sms, cudaStream_t s) {
  constexpr int rows = kRowWarps * (32 / LPR);
  const int64_t blocks = (p.num_tokens + rows - 1) / rows, cap = static_cast<int64_t>(num_sms) * 16;
  const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
  const int tile = (32 / LPR) * p.E * static_cast<int>(sizeof(T));
  const size_t smem = static_cast<size_t>(kRowWarps) * 2 * ((tile + 15) & ~15);
  // a warp's rows start on 16 bytes
  const int bulk = tile % 16 == 0 && (reinterpret_cast<uintptr_t>(p.grad_logits) & 15u) == 0;
  route_experts_backward_kernel<T, LPR><<<grid, kRowWarps * 32, smem, s>>>(p, bulk);
}

template <typename T>
void launch_backward(const RouteExpertsBackwardParams& p, int num_sms, cudaStream_t s) {
  if (p.scoring == 0 && !p.renormalize) {
    const int64_t blocks = (p.num_tokens + kFastWarps - 1) / kFastWarps;
    const int64_t cap = static_cast<int64_t>(num_sms) * 8;
    const unsigned grid = static_cast<unsigned>(blocks < cap ? blocks : cap);
    route_experts_backward_dense_kernel<T>
        <<<grid, kFastWarps * 32, sizeof(float) * kFastWarps * p.E, s>>>(p);
  } else if (p.k <= 8) {
    launch_backward_picks<T, 8>(p, num_sms, s);
  } else if (p.k <= 16) {
    launch_backward_picks<T, 16>(p, num_sms, s);
  } else {
    launch_backward_picks<T, 32>(p, num_sms, s);
  }
}
}  // namespace

bool route_experts_set_attributes() {
  const int most = kRowWarps * 2 * 4 * kRouteMaxExperts * 4;  // 64 KB: f32, eight lanes per row
  return cudaFuncSetAttribute(route_experts_backward_kernel<float, 8>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize, most) == cudaSuccess;
}

int launch_route_experts_backward(int dtype, const RouteExpertsBackwardParams& p, int num_sms,
                                  cudaStream_t s) {
  if (p.num_tokens <= 0) return 0;
  if (dtype == kF32) launch_backward<float>(p, num_sms, s);
  else if (dtype == kBF16) launch_backward<__nv_bfloat16>(p, num_sms, s);
  else launch_backward<__half>(p, num_sms, s);
  return 0;
}

}  // namespace cmoe
