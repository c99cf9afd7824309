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
// Packed layout: records [E][N/16][K/64], one per 16 n x 64 k: 512 bytes of nibbles, then for each
// group (two with G = 32, else one) 8 x 2 scales (n = gid, gid + 8) and, with zero points, 8 x 2
// bytes of them.  A column strip is one contiguous stream that holds all that its products
// need.  The nibbles are one 16-byte vector per lane (gid = lane / 4, tig = lane % 4), one
// 32-bit word per k16 step s, nibble i of its halves (h = 0, 1):
//     n = 16 tile + gid + 8 (i & 1),  k = 64 block + 32 (s >> 1) + 8 tig + 4 (s & 1) + 2 (i >> 1) + h
// This k order makes the activations of two steps 16 consecutive bytes per lane, and a pair of
// steps never leaves a group of 32.  The word is rotated left so that nibble 0 sits at the top
// of the mantissa.
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
__global__ void int4_pack_kernel(const uint8_t* __restrict__ q, int E, int K, int N, int rec,
                                 char* __restrict__ out) {
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
    *reinterpret_cast<uint32_t*>(out + (i >> 7) * rec + (i & 127) * 4) =
        __funnelshift_l(w, w, Nib<T>::kShift);
  }
}

// One thread per scale (and zero point) of a record.
__global__ void int4_pack_groups_kernel(const uint16_t* __restrict__ scales,
                                        const uint8_t* __restrict__ zeros, int E, int K, int N,
                                        int G, int rec, char* __restrict__ out) {
  const int per = G == 32 ? 2 : 1, kb = K / 64, nt = N / 16;
  const int64_t total = static_cast<int64_t>(E) * nt * kb * per * 16;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int r = static_cast<int>(i & 15), h = static_cast<int>(i >> 4) % per;
    const int64_t t = (i >> 4) / per;  // record
    const int b = static_cast<int>(t % kb), tile = static_cast<int>((t / kb) % nt);
    const int64_t e = t / kb / nt;
    const int n = tile * 16 + (r >> 1) + 8 * (r & 1);
    const int64_t from = (e * (K / G) + (64 * b + 32 * h) / G) * N + n;
    char* o = out + t * rec + 512;
    reinterpret_cast<uint16_t*>(o + 32 * h)[r] = scales[from];
    if (zeros) reinterpret_cast<uint8_t*>(o + 32 * per + 16 * h)[r] = zeros[from];
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
    int4_expand_kernel(const char* __restrict__ w, int rec, int per, bool zeros, int K, int N,
                       T* __restrict__ out) {
  using T2 = typename Pair<T>::type;
  constexpr int kCols = kTrans ? 64 : 128;
  constexpr int kPitch = kCols + 8;
  __shared__ alignas(16) T buf[(kTrans ? 128 : 64) * kPitch];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, gid = lane >> 2, tig = lane & 3;
  const int nb = N / 128, kb = K / 64;
  const int nblk = blockIdx.x % nb;
  const int b = (blockIdx.x / nb) % kb;
  const int64_t e = blockIdx.x / nb / kb;
  const int64_t tile = e * (N / 16) + nblk * 8 + warp;
  const char* record = w + (tile * kb + b) * rec;
  const uint4 q = __ldcs(reinterpret_cast<const uint4*>(record) + lane);
  const uint32_t word[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int hg = h & (per - 1);
    const T* scale = reinterpret_cast<const T*>(record + 512 + 32 * hg) + 2 * gid;
    const uint8_t* zero =
        reinterpret_cast<const uint8_t*>(record + 512 + 32 * per + 16 * hg) + 2 * gid;
    T2 sc[2], off[2];
#pragma unroll
    for (int r = 0; r < 2; ++r) {
      sc[r].x = sc[r].y = scale[r];
      off[r].x = off[r].y = Elem<T>::from_f(16.f + (zeros ? static_cast<float>(zero[r]) : 8.f));
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
constexpr int kMaxRecord = 608;  // int4_record_bytes(32, true)
constexpr int kStageBlocks = 2;  // k64 blocks of a ring stage

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N> __device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

// Expert of chunk c: the number of experts whose chunks all come before it.
__device__ __forceinline__ int find_expert(const int32_t* __restrict__ prefix, int E, int c) {
  int e = 0;
  for (int i = 0; i < E; i += 32) {
    const int at = i + (threadIdx.x & 31) + 1;
    e += __popc(__ballot_sync(0xffffffffu, at <= E && __ldg(prefix + at) <= c));
  }
  return e;
}

// A unit is (chunk of at most 8 NT rows of one expert, WN strips of 16 output columns); the warps
// of a CTA are WN strips x WK pieces of K, and the CTA takes every gridDim-th unit.  A warp
// streams the records of its piece through a ring of its own in shared memory (16-byte cp.async,
// kStages - 1 stages ahead, across units), so no warp waits for another except to add up the
// WK partial sums of a unit.  MATS = 2: gate and up.  kDown: rows are sorted rows of the
// intermediate, the result is weighted and goes to the (token, slot) row of the f32 slot
// buffer; else rows are tokens and the activation is applied.
template <typename T, int MATS, bool kDown, int NT, bool kG32>
__global__ void __launch_bounds__(kWarps * 32, NT <= 2 ? 2 : 1) int4_gemm_kernel(Int4Params p) {
  using T2 = typename Pair<T>::type;
  constexpr int kStages = MATS == 2 ? 4 : 6;
  constexpr int kRows = 8 * NT, kPitch = 20;  // partial sums [row][16 + 4]
  constexpr int kPer = kG32 ? 2 : 1;
  constexpr bool kOnes = NT == 1;
  extern __shared__ __align__(16) char smem[];
  float* red = reinterpret_cast<float*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int rec = p.rec;
  const int stage_bytes = MATS * kStageBlocks * rec;
  char* ring = smem + kWarps * MATS * kRows * kPitch * 4 + warp * kStages * stage_bytes;
  const uint32_t ring_addr = smem_addr(ring);
  const int wk = warp % p.wk, wn = warp / p.wk, wn_count = kWarps / p.wk;
  const int ntiles = p.N / 16, kb = p.K / 64;
  const int nunits = (ntiles + wn_count - 1) / wn_count;
  const int per = (kb + p.wk - 1) / p.wk;
  const int b0 = min(wk * per, kb), b1 = min(b0 + per, kb);
  const int nstages = (per + kStageBlocks - 1) / kStageBlocks;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  const int64_t units = static_cast<int64_t>(__ldg(p.chunk_prefix + p.E)) * nunits;

  // the ring's producer side: unit pu, stage ps
  int64_t pu = blockIdx.x;
  int ps = 0, slot_in = 0;
  int64_t strip = 0;  // first record of the strip
  auto locate = [&]() {
    if (pu < units) {
      const int c = static_cast<int>(pu / nunits);
      const int nt = static_cast<int>(pu % nunits) * wn_count + wn;
      strip = nt < ntiles
                  ? (static_cast<int64_t>(find_expert(p.chunk_prefix, p.E, c)) * ntiles + nt) * kb
                  : -1;
    }
  };
  auto issue = [&]() {
    if (pu < units) {
      const int b = b0 + ps * kStageBlocks;
      if (strip >= 0 && b < b1) {
        const int n16 = min(kStageBlocks, b1 - b) * rec / 16;
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const char* src = static_cast<const char*>(p.w[m]) + (strip + b) * rec;
          const uint32_t dst = ring_addr + slot_in * stage_bytes + m * kStageBlocks * rec;
          for (int i = lane; i < n16; i += 32) cp_async16(dst + i * 16, src + i * 16);
        }
      }
      if (++ps == nstages) {
        ps = 0;
        pu += gridDim.x;
        locate();
      }
    }
    cp_async_commit();
    slot_in = slot_in + 1 == kStages ? 0 : slot_in + 1;
  };
  locate();
#pragma unroll
  for (int i = 0; i < kStages - 1; ++i) issue();

  int slot = 0;
  for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = static_cast<int>(u / nunits);
    const int nt = static_cast<int>(u % nunits) * wn_count + wn;
    const int e = find_expert(p.chunk_prefix, p.E, c);
    const int row0 = __ldg(p.offsets + e) + (c - __ldg(p.chunk_prefix + e)) * kRows;
    const int rows = min(kRows, __ldg(p.offsets + e + 1) - row0);
    const T* xr[NT];
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const int r = 8 * j + gid;
      xr[j] = nullptr;
      if (r < rows)
        xr[j] = static_cast<const T*>(p.x) +
                static_cast<int64_t>(kDown ? row0 + r : __ldg(p.sorted_token + row0 + r)) * p.K +
                8 * tig;
    }
    const int tiles = (rows + 7) / 8;
    float fin[MATS][NT][4] = {};
    for (int st = 0; st < nstages; ++st) {
      const int b = b0 + st * kStageBlocks;
      const int blocks = nt < ntiles ? min(kStageBlocks, b1 - b) : 0;
      uint4 xv[kStageBlocks][NT][2];
      if (NT == 1) {  // few enough registers to have them under way before the wait
#pragma unroll
        for (int i = 0; i < kStageBlocks; ++i)
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            xv[i][0][h] = make_uint4(0, 0, 0, 0);
            if (i < blocks && xr[0])
              xv[i][0][h] = *reinterpret_cast<const uint4*>(xr[0] + 64 * (b + i) + 32 * h);
          }
      }
      cp_async_wait<kStages - 2>();
      __syncwarp();
      const char* stage = ring + slot * stage_bytes;
#pragma unroll
      for (int i = 0; i < kStageBlocks; ++i) {
        if (i >= blocks) break;
        if (NT > 1) {
#pragma unroll
          for (int j = 0; j < NT; ++j)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
              xv[i][j][h] = make_uint4(0, 0, 0, 0);
              if (j < tiles && xr[j])
                xv[i][j][h] = *reinterpret_cast<const uint4*>(xr[j] + 64 * (b + i) + 32 * h);
            }
        }
        float xs[kPer][4] = {};
        if (kOnes) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {
            const uint4 v = xv[i][0][h];
            mma16816<T>(xs[h & (kPer - 1)], Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne,
                        v.x, v.y);
            mma16816<T>(xs[h & (kPer - 1)], Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne, Nib<T>::kOne,
                        v.z, v.w);
          }
        }
#pragma unroll
        for (int m = 0; m < MATS; ++m) {
          const char* record = stage + (m * kStageBlocks + i) * rec;
          const uint4 wq = *(reinterpret_cast<const uint4*>(record) + lane);
          const uint32_t word[4] = {wq.x, wq.y, wq.z, wq.w};
          float acc[NT][4];
#pragma unroll
          for (int s = 0; s < 4; ++s) {
            const int hg = (s >> 1) & (kPer - 1);
            float z0 = 24.f, z1 = 24.f;
            if (p.zeros) {
              const uint8_t* zp =
                  reinterpret_cast<const uint8_t*>(record + 512 + 32 * kPer + 16 * hg) + 2 * gid;
              z0 = 16.f + static_cast<float>(zp[0]);
              z1 = 16.f + static_cast<float>(zp[1]);
            }
            uint32_t a[4];
#pragma unroll
            for (int f = 0; f < 4; ++f) {
              a[f] = nib_pair<T>(word[s], f);
              if (!kOnes) {  // q - z, exact
                T2 off;
                off.x = off.y = Elem<T>::from_f((f & 1) ? z1 : z0);
                const T2 v = __hsub2(*reinterpret_cast<const T2*>(&a[f]), off);
                a[f] = *reinterpret_cast<const uint32_t*>(&v);
              }
            }
            const bool first = s == 0 || (kG32 && s == 2), last = s == 3 || (kG32 && s == 1);
#pragma unroll
            for (int j = 0; j < NT; ++j) {
              if (NT > 1 && j >= tiles) break;
              if (first) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.f;
              const uint4 v = xv[i][j][s >> 1];
              mma16816<T>(acc[j], a[0], a[1], a[2], a[3], (s & 1) ? v.z : v.x, (s & 1) ? v.w : v.y);
            }
            if (last) {
              const T2 sc = *(reinterpret_cast<const T2*>(record + 512 + 32 * hg) + gid);
              const float s0 = Elem<T>::to_f(sc.x), s1 = Elem<T>::to_f(sc.y);
#pragma unroll
              for (int j = 0; j < NT; ++j) {
                if (NT > 1 && j >= tiles) break;
                if (kOnes) {
                  acc[j][0] -= z0 * xs[hg][0];
                  acc[j][1] -= z0 * xs[hg][1];
                  acc[j][2] -= z1 * xs[hg][0];
                  acc[j][3] -= z1 * xs[hg][1];
                }
                fin[m][j][0] += s0 * acc[j][0];
                fin[m][j][1] += s0 * acc[j][1];
                fin[m][j][2] += s1 * acc[j][2];
                fin[m][j][3] += s1 * acc[j][3];
              }
            }
          }
        }
      }
      __syncwarp();
      issue();
      slot = slot + 1 == kStages ? 0 : slot + 1;
    }
#pragma unroll
    for (int m = 0; m < MATS; ++m)
#pragma unroll
      for (int j = 0; j < NT; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          red[((warp * MATS + m) * kRows + 8 * j + 2 * tig + (i & 1)) * kPitch + gid +
              8 * (i >> 1)] = fin[m][j][i];
    __syncthreads();
    for (int i = threadIdx.x; i < wn_count * rows * 16; i += kWarps * 32) {
      const int n = i & 15, r = (i >> 4) % rows, w = (i >> 4) / rows;
      const int col = (static_cast<int>(u % nunits) * wn_count + w) * 16 + n;
      if (col >= p.N) continue;
      float v = 0.f, v1 = 0.f;
      for (int q = 0; q < p.wk; ++q) {  // in the order of k
        const float* from = red + ((w * p.wk + q) * MATS * kRows + r) * kPitch + n;
        v += from[0];
        if (MATS == 2) v1 += from[kRows * kPitch];
      }
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
  cp_async_wait<0>();
}

// out[t] = sum over the token's slots in slot order, one rounding.
template <typename T>
__global__ void int4_combine_kernel(const float* __restrict__ slots, const uint32_t* __restrict__ idx,
                                    int64_t T_, int k, int H, int E, T* __restrict__ out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
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

// Launched as a programmatic dependent: waits for the kernel before it with griddepcontrol.wait.
template <typename... Args>
bool launch_dependent(void (*kernel)(Args...), int grid, int threads, size_t smem, cudaStream_t s,
                      Args... args) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(static_cast<unsigned>(threads));
  cfg.dynamicSmemBytes = smem;
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, args...) == cudaSuccess;
}

// Pieces of K: as many as leave a warp three k64 blocks or more.
int pieces_of(int K) {
  int wk = kWarps;
  while (wk > 1 && K / 64 < 3 * wk) wk /= 2;
  return wk;
}

template <typename T, int MATS, bool kDown, int NT, bool kG32>
struct Gemm {
  static constexpr auto kernel = int4_gemm_kernel<T, MATS, kDown, NT, kG32>;
  static size_t smem(int rec) {
    return static_cast<size_t>(kWarps) *
           (MATS * 8 * NT * 20 * 4 + (MATS == 2 ? 4 : 6) * MATS * kStageBlocks * rec);
  }
  static bool attributes() {
    return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                static_cast<int>(smem(kMaxRecord))) == cudaSuccess;
  }
  static bool launch(Int4Params p, int num_sms, cudaStream_t s) {
    p.wk = pieces_of(p.K);
    // resident CTAs: two on an SM where registers and shared memory allow (227 KB, 1 KB a CTA)
    const size_t bytes = smem(p.rec);
    const int per_sm = NT <= 2 && 2 * (bytes + 1024) <= 227 * 1024 ? 2 : 1;
    return launch_dependent(kernel, num_sms * per_sm, kWarps * 32, bytes, s, p);
  }
};

template <typename T, int NT, bool kG32>
bool launch_gemms(const Int4Params& g1, const Int4Params& g2, int num_sms, cudaStream_t s) {
  const bool ok = g1.w[1] ? Gemm<T, 2, false, NT, kG32>::launch(g1, num_sms, s)
                          : Gemm<T, 1, false, NT, kG32>::launch(g1, num_sms, s);
  return ok && Gemm<T, 1, true, NT, kG32>::launch(g2, num_sms, s);
}

template <typename T, int NT, bool kG32> bool gemm_attributes() {
  return Gemm<T, 2, false, NT, kG32>::attributes() && Gemm<T, 1, false, NT, kG32>::attributes() &&
         Gemm<T, 1, true, NT, kG32>::attributes();
}
template <typename T> bool gemm_attributes() {
  return gemm_attributes<T, 1, false>() && gemm_attributes<T, 2, false>() &&
         gemm_attributes<T, 4, false>() && gemm_attributes<T, 1, true>() &&
         gemm_attributes<T, 2, true>() && gemm_attributes<T, 4, true>();
}

template <typename T>
bool launch_ffn(int nt, const Int4Params& g1, const Int4Params& g2, const uint32_t* idx,
                int64_t T_, int k, void* out, int num_sms, cudaStream_t s) {
  bool ok;
  if (g1.G == 32)
    ok = nt == 1   ? launch_gemms<T, 1, true>(g1, g2, num_sms, s)
         : nt == 2 ? launch_gemms<T, 2, true>(g1, g2, num_sms, s)
                   : launch_gemms<T, 4, true>(g1, g2, num_sms, s);
  else
    ok = nt == 1   ? launch_gemms<T, 1, false>(g1, g2, num_sms, s)
         : nt == 2 ? launch_gemms<T, 2, false>(g1, g2, num_sms, s)
                   : launch_gemms<T, 4, false>(g1, g2, num_sms, s);
  return ok && launch_dependent(int4_combine_kernel<T>, grid_for(T_ * g2.N, num_sms), 256, 0, s,
                                static_cast<const float*>(g2.out), idx, T_, k, g2.N, g2.E,
                                static_cast<T*>(out));
}

template <typename T>
void expand(const void* w, int E, int K, int N, int G, bool zeros, bool trans, void* out,
            cudaStream_t s) {
  const unsigned grid = static_cast<unsigned>(static_cast<int64_t>(E) * (K / 64) * (N / 128));
  const int rec = int4_record_bytes(G, zeros), per = G == 32 ? 2 : 1;
  const char* from = static_cast<const char*>(w);
  T* to = static_cast<T*>(out);
  if (trans)
    int4_expand_kernel<T, true><<<grid, 256, 0, s>>>(from, rec, per, zeros, K, N, to);
  else
    int4_expand_kernel<T, false><<<grid, 256, 0, s>>>(from, rec, per, zeros, K, N, to);
}

}  // namespace

int int4_record_bytes(int G, bool zeros) { return 512 + (G == 32 ? 2 : 1) * (zeros ? 48 : 32); }

bool int4_set_attributes() { return gemm_attributes<__nv_bfloat16>() && gemm_attributes<__half>(); }

void launch_int4_expand(int dtype, const void* w, int E, int K, int N, int G, bool zeros,
                        bool trans, void* out, cudaStream_t s) {
  if (dtype == kBF16) expand<__nv_bfloat16>(w, E, K, N, G, zeros, trans, out, s);
  else expand<__half>(w, E, K, N, G, zeros, trans, out, s);
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
                     int K, int N, int G, void* packed, int num_sms, cudaStream_t s) {
  char* base = static_cast<char*>(packed);
  const int rec = int4_record_bytes(G, zeros != nullptr);
  const int grid = grid_for(static_cast<int64_t>(E) * K * N / 8, num_sms);
  if (dtype == kBF16) int4_pack_kernel<__nv_bfloat16><<<grid, 256, 0, s>>>(q, E, K, N, rec, base);
  else int4_pack_kernel<__half><<<grid, 256, 0, s>>>(q, E, K, N, rec, base);
  int4_pack_groups_kernel<<<grid_for(static_cast<int64_t>(E) * (K / 32) * N, num_sms), 256, 0, s>>>(
      static_cast<const uint16_t*>(scales), zeros, E, K, N, G, rec, base);
  return 2;
}

int launch_int4_ffn(int dtype, int chunk_rows, const Int4Params& g1, const Int4Params& g2,
                    const uint32_t* idx, int64_t num_tokens, int k, void* out, int num_sms,
                    cudaStream_t s) {
  const bool ok =
      dtype == kBF16
          ? launch_ffn<__nv_bfloat16>(chunk_rows / 8, g1, g2, idx, num_tokens, k, out, num_sms, s)
          : launch_ffn<__half>(chunk_rows / 8, g1, g2, idx, num_tokens, k, out, num_sms, s);
  return ok ? 3 : 0;
}

}  // namespace cmoe
