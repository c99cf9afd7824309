// Q: the expert FFN on 4-bit weights with group scales.
//
// A weight matrix W [E, K, N] (K the reduction) is held as q in 0..15 with one scale, and
// optionally one zero point (else 8), per group of G consecutive k and column n:
//     W[e,k,n] = (q[e,k,n] - z[e,k/G,n]) * s[e,k/G,n]
// and the layer is y_t = sum_j w_tj (act(x_t Gate_e) * (x_t Up_e)) Down_e  (or act(x_t Gate_e)
// Down_e without Up), e = idx[t,j], ids >= E skipped.
//
// The products run on mma.sync m16n8k16 with the weights as the 16-row operand: a call of few
// tokens streams weights, and that fragment can be made from packed nibbles in registers, so the
// weights go from memory to the tensor cores without touching shared memory.  For a group,
//     sum_k W x = s * (sum_k (16 + q) x - (16 + z) * sum_k x)
// where 16 + q is exact in bf16 and f16 and one LOP3 away from the nibble (the nibble is the top
// of the mantissa of a number in [16, 32)); sum_k x comes from one more product with a matrix of
// ones.  The products are exact, so the scales and zero points act on f32 sums: no weight is
// ever rounded.
//
// Packed layout: tiles of 16 n x 64 k, 512 bytes, ordered [E][N/16][K/64], one 16-byte vector
// per lane (gid = lane / 4, tig = lane % 4), one 32-bit word per k16 step s, nibble i of its
// halves (h = 0, 1):
//     n = 16 tile + gid + 8 (i & 1),  k = 64 block + 32 (s >> 1) + 8 tig + 4 (s & 1) + 2 (i >> 1) + h
// This k order makes the activations of two steps 16 consecutive bytes per lane, and a step
// never leaves a group of 32.  The word is rotated left so that nibble 0 sits at the top of the
// mantissa.  Scales are [E][N/16][K/G][8][2] (n = gid, gid + 8), zero points likewise in bytes.
#include <stdint.h>

#include "common.cuh"
#include "kernels.h"

namespace cmoe {

namespace {

template <typename T> struct Nib;
template <> struct Nib<__nv_bfloat16> {
  static constexpr int kShift = 3;  // 7 mantissa bits
  static constexpr uint32_t kMask = 0x00780078u, kMagic = 0x41804180u, kOne = 0x3f803f80u;
};
template <> struct Nib<__half> {
  static constexpr int kShift = 6;  // 10 mantissa bits
  static constexpr uint32_t kMask = 0x03c003c0u, kMagic = 0x4c004c00u, kOne = 0x3c003c00u;
};

__device__ __forceinline__ uint32_t rotr(uint32_t v, int n) { return __funnelshift_r(v, v, n); }

// Fragment register i of a packed word: the pair (16 + q_lo, 16 + q_hi).
template <typename T> __device__ __forceinline__ uint32_t nib_pair(uint32_t w, int i) {
  return (rotr(w, 4 * i) & Nib<T>::kMask) | Nib<T>::kMagic;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                        uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                 uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// ---- quantisation and packing (once per set of weights) --------------------------------------

// One thread per (expert, group, column): min / max over the group's k, then the nibbles.
template <typename T>
__global__ void int4_quantize_kernel(const T* __restrict__ w, int E, int K, int N, int G,
                                     int symmetric, uint8_t* __restrict__ q, T* __restrict__ scales,
                                     uint8_t* __restrict__ zeros) {
  const int64_t total = static_cast<int64_t>(E) * (K / G) * N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int n = static_cast<int>(i % N);
    const int64_t eg = i / N;  // e * K/G + group; its first row of w is eg * G
    const T* p = w + eg * G * N + n;
    float lo = 0.f, hi = 0.f;
    for (int k = 0; k < G; ++k) {
      const float v = Elem<T>::to_f(p[static_cast<int64_t>(k) * N]);
      lo = fminf(lo, v);
      hi = fmaxf(hi, v);
    }
    const T st = Elem<T>::from_f(symmetric ? __fdiv_rn(fmaxf(-lo, hi), 7.f)
                                           : __fdiv_rn(hi - lo, 15.f));
    const float s = Elem<T>::to_f(st);
    float z = 8.f;
    if (!symmetric) z = s > 0.f ? fminf(fmaxf(rintf(__fdiv_rn(-lo, s)), 0.f), 15.f) : 0.f;
    scales[i] = st;
    if (zeros) zeros[i] = static_cast<uint8_t>(z);
    uint8_t* o = q + eg * (G / 2) * N + n;
    for (int k = 0; k < G; k += 2) {
      uint32_t b = 0;
      for (int h = 0; h < 2; ++h) {
        const float v = Elem<T>::to_f(p[static_cast<int64_t>(k + h) * N]);
        const float r = s > 0.f ? rintf(__fdiv_rn(v, s)) + z : z;
        b |= static_cast<uint32_t>(fminf(fmaxf(r, 0.f), 15.f)) << (4 * h);
      }
      o[static_cast<int64_t>(k / 2) * N] = static_cast<uint8_t>(b);
    }
  }
}

// One thread per packed 32-bit word.
template <typename T>
__global__ void int4_pack_kernel(const uint8_t* __restrict__ q, int E, int K, int N,
                                 uint32_t* __restrict__ out) {
  const int nt = N / 16, kb = K / 64;
  const int64_t total = static_cast<int64_t>(E) * nt * kb * 128;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int s = static_cast<int>(i & 3), lane = static_cast<int>(i >> 2) & 31;
    int64_t t = i >> 7;
    const int b = static_cast<int>(t % kb);
    t /= kb;
    const int n0 = static_cast<int>(t % nt) * 16;
    const int64_t e = t / nt;
    const int gid = lane >> 2, tig = lane & 3;
    uint32_t w = 0;
    for (int f = 0; f < 4; ++f) {
      const int n = n0 + gid + 8 * (f & 1);
      const int k = 64 * b + 32 * (s >> 1) + 8 * tig + 4 * (s & 1) + 2 * (f >> 1);
      const uint32_t two = q[(e * (K / 2) + k / 2) * N + n];  // k even: low nibble k, high k + 1
      w |= (two & 15u) << (4 * f);
      w |= (two >> 4) << (16 + 4 * f);
    }
    out[i] = __funnelshift_l(w, w, Nib<T>::kShift);
  }
}

// [E][K/G][N] -> [E][N/16][K/G][8][2]
template <typename V>
__global__ void int4_pack_groups_kernel(const V* __restrict__ in, int E, int KG, int N,
                                        V* __restrict__ out) {
  const int64_t total = static_cast<int64_t>(E) * KG * N;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int r = static_cast<int>(i & 15);
    int64_t t = i >> 4;
    const int g = static_cast<int>(t % KG);
    t /= KG;
    const int n = static_cast<int>(t % (N / 16)) * 16 + (r >> 1) + 8 * (r & 1);
    const int64_t e = t / (N / 16);
    out[i] = in[(e * KG + g) * N + n];
  }
}

// ---- weights back in 16 bits (for calls of many rows) --------------------------------------------

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

// One CTA per (expert, 64 k, 128 n): a warp takes 16 n (one packed tile), the rows leave through
// shared memory in 256-byte (out [E,K,N]) or 128-byte (kTrans: out [E,N,K]) pieces.  q - z is
// exact, the product with the scale is rounded once.
template <typename T, bool kTrans>
__global__ void __launch_bounds__(256)
    int4_expand_kernel(const uint4* __restrict__ w, const T* __restrict__ scale,
                       const uint8_t* __restrict__ zero, int K, int N, int G, T* __restrict__ out) {
  using T2 = typename Pair<T>::type;
  constexpr int kCols = kTrans ? 64 : 128;
  constexpr int kPitch = kCols + 8;
  __shared__ alignas(16) T buf[(kTrans ? 128 : 64) * kPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int nb = N / 128, kb = K / 64, kg = K / G;
  const int nblk = blockIdx.x % nb;
  const int b = (blockIdx.x / nb) % kb;
  const int64_t e = blockIdx.x / nb / kb;
  const int64_t tile = e * (N / 16) + nblk * 8 + warp;
  const uint4 q = __ldcs(w + (tile * kb + b) * 32 + lane);
  const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int64_t gi = ((tile * kg + (64 * b + 32 * h) / G) * 8 + gid) * 2;
    T2 sc[2], off[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sc[r].x = sc[r].y = scale[gi + r];
      off[r].x = off[r].y =
          Elem<T>::from_f(16.f + (zero ? static_cast<float>(zero[gi + r]) : 8.f));
    }
#pragma unroll
    for (int s = 0; s < 2; ++s)
#pragma unroll
      for (int f = 0; f < 4; ++f) {
        const uint32_t u = nib_pair<T>(word[2 * h + s], f);
        const T2 v = __hmul2(__hsub2(*reinterpret_cast<const T2*>(&u), off[f & 1]), sc[f & 1]);
        const int n = 16 * warp + gid + 8 * (f & 1);
        const int k = 32 * h + 8 * tig + 4 * s + 2 * (f >> 1);
        if (kTrans) {
          *reinterpret_cast<T2*>(buf + n * kPitch + k) = v;
        } else {
          buf[k * kPitch + n] = v.x;
          buf[(k + 1) * kPitch + n] = v.y;
        }
      }
  }
  __syncthreads();
  constexpr int kVecs = kCols / 8;
  const int64_t row0 = kTrans ? e * N + nblk * 128 : e * K + b * 64;
  const int ld = kTrans ? K : N, col0 = kTrans ? b * 64 : nblk * 128;
#pragma unroll
  for (int i = threadIdx.x; i < 128 * 64 / 8; i += 256) {
    const int r = i / kVecs, c = (i % kVecs) * 8;
    *reinterpret_cast<uint4*>(out + (row0 + r) * ld + col0 + c) =
        *reinterpret_cast<const uint4*>(buf + r * kPitch + c);
  }
}

// ---- the products ------------------------------------------------------------------------------

constexpr int kWarps = 8;

__device__ __forceinline__ int find_expert(const int32_t* __restrict__ prefix, int E, int c) {
  int lo = 0, hi = E;  // prefix[lo] <= c < prefix[hi]
  while (hi - lo > 1) {
    const int mid = (lo + hi) >> 1;
    if (__ldg(prefix + mid) <= c) lo = mid;
    else hi = mid;
  }
  return lo;
}

// One CTA per (chunk of at most 8 NT rows of one expert, 16 output columns); its warps split K.
// MATS = 2: gate and up.  kDown: rows are sorted rows of the intermediate, the result is weighted
// and goes to the (token, slot) row of the f32 slot buffer; else rows are tokens and the
// activation is applied.
template <typename T, int MATS, bool kDown, int NT>
__global__ void __launch_bounds__(kWarps * 32) int4_gemm_kernel(Int4Params p) {
  __shared__ float red[kWarps][MATS][16][8 * NT + 1];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int ntiles = p.N / 16, kb = p.K / 64, kg = p.K / p.G;
  const int64_t units = static_cast<int64_t>(__ldg(p.chunk_prefix + p.E)) * ntiles;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = static_cast<int>(u / ntiles), nt = static_cast<int>(u % ntiles);
    const int e = find_expert(p.chunk_prefix, p.E, c);
    const int row0 = __ldg(p.offsets + e) + (c - __ldg(p.chunk_prefix + e)) * 8 * NT;
    const int rows = min(8 * NT, __ldg(p.offsets + e + 1) - row0);
    const T* xr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = 8 * j + gid;
      xr[j] = nullptr;
      if (r < rows)
        xr[j] = static_cast<const T*>(p.x) +
                static_cast<int64_t>(kDown ? row0 + r : __ldg(p.sorted_token + row0 + r)) * p.K;
    }
    const int64_t tile = static_cast<int64_t>(e) * ntiles + nt;
    float fin[MATS][NT][4] = {};
    for (int b = warp; b < kb; b += kWarps) {
      uint4 wq[MATS];
#pragma unroll
      for (int m = 0; m < MATS; ++m)
        wq[m] = __ldg(reinterpret_cast<const uint4*>(p.w[m]) + (tile * kb + b) * 32 + lane);
      uint4 xv[NT][2];
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int h = 0; h < 2; ++h)
          xv[j][h] = xr[j] ? *reinterpret_cast<const uint4*>(xr[j] + 64 * b + 32 * h + 8 * tig)
                           : make_uint4(0, 0, 0, 0);
#pragma unroll
      for (int h = 0; h < 2; ++h) {  // 32 k: never more than one group
        const int g = (64 * b + 32 * h) / p.G;
        float xs[NT][4] = {};
#pragma unroll
        for (int j = 0; j < NT; ++j) {
          mma16816<T>(xs[j], Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, xv[j][h].x,
                      xv[j][h].y);
          mma16816<T>(xs[j], Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, xv[j][h].z,
                      xv[j][h].w);
        }
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const uint32_t w0 = h ? wq[m].z : wq[m].x, w1 = h ? wq[m].w : wq[m].y;
          float acc[NT][4] = {};
          const uint32_t a0 = nib_pair<T>(w0, 0), a1 = nib_pair<T>(w0, 1),
                         a2 = nib_pair<T>(w0, 2), a3 = nib_pair<T>(w0, 3);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            mma16816<T>(acc[j], a0, a1, a2, a3, xv[j][h].x, xv[j][h].y);
          const uint32_t b0 = nib_pair<T>(w1, 0), b1 = nib_pair<T>(w1, 1),
                         b2 = nib_pair<T>(w1, 2), b3 = nib_pair<T>(w1, 3);
#pragma unroll
          for (int j = 0; j < NT; ++j)
            mma16816<T>(acc[j], b0, b1, b2, b3, xv[j][h].z, xv[j][h].w);
          const int64_t gi = ((tile * kg + g) * 8 + gid) * 2;
          const T* sp = static_cast<const T*>(p.scale[m]) + gi;
          const float s0 = Elem<T>::to_f(sp[0]), s1 = Elem<T>::to_f(sp[1]);
          float z0 = 24.f, z1 = 24.f;
          if (p.zero[m]) {
            z0 = 16.f + static_cast<float>(p.zero[m][gi]);
            z1 = 16.f + static_cast<float>(p.zero[m][gi + 1]);
          }
#pragma unroll
          for (int j = 0; j < NT; ++j) {
            fin[m][j][0] += s0 * (acc[j][0] - z0 * xs[j][0]);
            fin[m][j][1] += s0 * (acc[j][1] - z0 * xs[j][1]);
            fin[m][j][2] += s1 * (acc[j][2] - z1 * xs[j][0]);
            fin[m][j][3] += s1 * (acc[j][3] - z1 * xs[j][1]);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[warp][m][gid + 8 * (i >> 1)][8 * j + 2 * tig + (i & 1)] = fin[m][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < 16 * rows; i += blockDim.x) {
      const int n = i & 15, r = i >> 4;
      float v = 0.f, v1 = 0.f;
      for (int w = 0; w < kWarps; ++w) {
        v += red[w][0][n][r];
        if (MATS == 2) v1 += red[w][MATS - 1][n][r];
      }
      const int col = nt * 16 + n;
      if (kDown) {
        static_cast<float*>(p.out)[static_cast<int64_t>(__ldg(p.sorted_flat + row0 + r)) * p.N +
                                   col] = v * __ldg(p.sorted_w + row0 + r);
      } else {
        v = act_apply(v, p.act);
        if (MATS == 2) v *= v1;
        // the intermediate is rounded to the 16-bit type that the second product reads
        static_cast<T*>(p.out)[static_cast<int64_t>(row0 + r) * p.N + col] = Elem<T>::from_f(v);
      }
    }
    __syncthreads();
  }
}

// out[t] = sum over the token's slots in slot order, one rounding.
template <typename T>
__global__ void int4_combine_kernel(const float* __restrict__ slots, const uint32_t* __restrict__ idx,
                                    int64_t T_, int k, int H, int E, T* __restrict__ out) {
  const int64_t total = T_ * H;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / H;
    const int h = static_cast<int>(i % H);
    float v = 0.f;
    for (int j = 0; j < k; ++j)
      if (__ldg(idx + t * k + j) < static_cast<uint32_t>(E)) v += slots[(t * k + j) * H + h];
    out[i] = Elem<T>::from_f(v);
  }
}

int grid_for(int64_t n, int num_sms) {
  const int64_t b = (n + 255) / 256, cap = static_cast<int64_t>(num_sms) * 16;
  return static_cast<int>(b < cap ? b : cap);
}

template <typename T, int NT>
void launch_gemms(const Int4Params& g1, const Int4Params& g2, int grid, cudaStream_t s) {
  if (g1.w[1]) int4_gemm_kernel<T, 2, false, NT><<<grid, kWarps * 32, 0, s>>>(g1);
  else int4_gemm_kernel<T, 1, false, NT><<<grid, kWarps * 32, 0, s>>>(g1);
  int4_gemm_kernel<T, 1, true, NT><<<grid, kWarps * 32, 0, s>>>(g2);
}

template <typename T>
void launch_ffn(int nt, const Int4Params& g1, const Int4Params& g2, const uint32_t* idx,
                int64_t T_, int k, void* out, int num_sms, cudaStream_t s) {
  const int grid = num_sms * 4;
  if (nt == 1) launch_gemms<T, 1>(g1, g2, grid, s);
  else if (nt == 2) launch_gemms<T, 2>(g1, g2, grid, s);
  else launch_gemms<T, 4>(g1, g2, grid, s);
  int4_combine_kernel<T><<<grid_for(T_ * g2.N, num_sms), 256, 0, s>>>(
      static_cast<const float*>(g2.out), idx, T_, k, g2.N, g2.E, static_cast<T*>(out));
}

template <typename T>
void expand(const void* w, const void* scale, const uint8_t* zero, int E, int K, int N, int G,
            bool trans, void* out, cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(E) * (K / 64) * (N / 128));
  if (trans)
    int4_expand_kernel<T, true><<<grid, 256, 0, s>>>(static_cast<const uint4*>(w),
                                                     static_cast<const T*>(scale), zero, K, N, G,
                                                     static_cast<T*>(out));
  else
    int4_expand_kernel<T, false><<<grid, 256, 0, s>>>(static_cast<const uint4*>(w),
                                                      static_cast<const T*>(scale), zero, K, N, G,
                                                      static_cast<T*>(out));
}

}  // namespace

void launch_int4_expand(int dtype, const void* w, const void* scale, const uint8_t* zero, int E,
                        int K, int N, int G, bool trans, void* out, cudaStream_t s) {
  if (dtype == kBF16) expand<__nv_bfloat16>(w, scale, zero, E, K, N, G, trans, out, s);
  else expand<__half>(w, scale, zero, E, K, N, G, trans, out, s);
}

int int4_chunk_rows(int64_t rows, int E) {
  const int64_t per = rows / E;
  return per <= 6 ? 8 : per <= 12 ? 16 : 32;
}

int launch_int4_quantize(int dtype, const void* w, int E, int K, int N, int G, int symmetric,
                         uint8_t* q, void* scales, uint8_t* zeros, int num_sms, cudaStream_t s) {
  const int grid = grid_for(static_cast<int64_t>(E) * (K / G) * N, num_sms);
  if (dtype == kBF16)
    int4_quantize_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(
        static_cast<const __nv_bfloat16*>(w), E, K, N, G, symmetric, q,
        static_cast<__nv_bfloat16*>(scales), zeros);
  else
    int4_quantize_kernel<__half><<<grid, 256, 0, s>>>(static_cast<const __half*>(w), E, K, N, G,
                                                      symmetric, q, static_cast<__half*>(scales),
                                                      zeros);
  return 0;
}

int launch_int4_pack(int dtype, const uint8_t* q, const void* scales, const uint8_t* zeros, int E,
                     int K, int N, int G, const Int4Layout& L, void* packed, int num_sms,
                     cudaStream_t s) {
  char* base = static_cast<char*>(packed);
  const int grid = grid_for(static_cast<int64_t>(E) * K * N / 8, num_sms);
  uint32_t* words = reinterpret_cast<uint32_t*>(base);
  if (dtype == kBF16) int4_pack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(q, E, K, N, words);
  else int4_pack_kernel<__half><<<grid, 256, 0, s>>>(q, E, K, N, words);
  const int gg = grid_for(static_cast<int64_t>(E) * (K / G) * N, num_sms);
  int4_pack_groups_kernel<uint16_t><<<gg, 256, 0, s>>>(static_cast<const uint16_t*>(scales), E,
                                                       K / G, N,
                                                       reinterpret_cast<uint16_t*>(base + L.scales));
  if (zeros)
    int4_pack_groups_kernel<uint8_t><<<gg, 256, 0, s>>>(
        zeros, E, K / G, N, reinterpret_cast<uint8_t*>(base + L.zeros));
  return zeros ? 3 : 2;
}

int launch_int4_ffn(int dtype, int chunk_rows, const Int4Params& g1, const Int4Params& g2,
                    const uint32_t* idx, int64_t num_tokens, int k, void* out, int num_sms,
                    cudaStream_t s) {
  if (dtype == kBF16)
    launch_ffn<__nv_bfloat16>(chunk_rows / 8, g1, g2, idx, num_tokens, k, out, num_sms, s);
  else
    launch_ffn<__half>(chunk_rows / 8, g1, g2, idx, num_tokens, k, out, num_sms, s);
  return 3;
}

}  // namespace cmoe
