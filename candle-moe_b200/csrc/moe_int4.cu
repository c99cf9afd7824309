// Q: the expert FFN on 4-bit weights with group scales.
//
// A weight matrix W [E, K, N] (K the reduction) is held as q in 0..15 with one scale, and
// optionally one zero point (else 8), per group of G consecutive k and column n:
//     W[e,k,n] = (q[e,k,n] - z[e,k/G,n]) * s[e,k/G,n]
// and the layer is y_t = sum_j w_tj (act(x_t Gate_e) * (x_t Up_e)) Down_e  (or act(x_t Gate_e)
// Down_e without Up), e = idx[t,j], ids >= E skipped.
//
// Three paths, by the rows (token, slot) of the call:
//   - at most 48: the kernels below, on mma.sync m16n8k16 with the weights as the 16-row operand.
//     Such a call streams weights, and that fragment is made from packed nibbles in registers:
//         sum_k W x = s * (sum_k (16 + q) x - (16 + z) * sum_k x)      (k over a group)
//     where 16 + q is exact in bf16 and f16 and one LOP3 away from the nibble (the top of the
//     mantissa of a number in [16, 32)), and sum_k x comes from one more product with a matrix
//     of ones.  The products are exact and the scales and zero points act on f32 sums: no
//     weight is rounded.
//   - more: moe_int4_mma.cu, tcgen05 with the unpacked weights in tensor memory.
//   - from 384 rows per expert on: int4_expand_kernel writes the weights in 16 bits once, and the
//     grouped GEMMs of the 16-bit experts run on them.
// Measured (mean of a run of calls, inputs larger than L2): 128 experts of 2048 x 768, top 8: one
// token 15 us (19 MB of weights and scales; floor 3), 8 tokens 50, 512 tokens 146 (316 MB; floor
// 48), 2048 tokens 339; 8 experts of 4096 x 1536, top 2, 8 tokens 32 us (71 MB; floor 11).
//
// Packed layout: records [E][N/16][K/64], one per 16 n x 64 k: 512 bytes of nibbles, then for each
// group (two with G = 32, else one) 8 x 2 scales (n = gid, gid + 8) and, with zero points, 8 x 2
// bytes of them.  A column strip is one contiguous stream that holds all that its products
// need.  The nibbles are one 16-byte vector per lane (gid = lane / 4, tig = lane % 4), one
// 32-bit word per k16 step s, nibble i of its halves (h = 0, 1) as the fragment has it:
//     n = 16 tile + gid + 8 (i & 1),  k = 64 block + 16 s + 8 (i >> 1) + 2 tig + h
// The word is rotated left so that nibble 0 sits at the top of the mantissa.
#include <stdint.h>

#include "common.cuh"
#include "int4.cuh"
#include "kernels.h"

namespace cmoe {

namespace {

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                         uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                        uint32_t a2, uint32_t a3, uint32_t b0,
                                                        uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                 uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The same with a zero accumulator.
template <typename T>
__device__ __forceinline__ void mma16816_zero(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2,
                                              uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816_zero<__nv_bfloat16>(float (&d)[4], uint32_t a0,
                                                             uint32_t a1, uint32_t a2, uint32_t a3,
                                                             uint32_t b0, uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
}
template <>
__device__ __forceinline__ void mma16816_zero<__half>(float (&d)[4], uint32_t a0, uint32_t a1,
                                                      uint32_t a2, uint32_t a3, uint32_t b0,
                                                      uint32_t b1) {
  asm(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, "
      "{%10,%10,%10,%10};"
      : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
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
      const int k = 64 * b + 16 * s + 8 * (f >> 1) + 2 * tig;
      const uint32_t two = q[(e * (K / 2) + k / 2) * N + n];  // k even: low nibble k, high k + 1
      w |= (two & 15u) << (4 * f);
      w |= (two >> 4) << (16 + 4 * f);
    }
    *reinterpret_cast<uint32_t*>(out + (i >> 7) * rec + (i & 127) * 4) =
        __funnelshift_l(w, w, Nib<T>::kShift);
  }
}

// One thread per scale (and zero point) of a record.  A zero point is its low four bits, so that
// the kernels, which read them in different ways, see the same number.
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
    if (zeros) reinterpret_cast<uint8_t*>(o + 32 * per + 16 * h)[r] = zeros[from] & 15u;
  }
}

// ---- weights back in 16 bits (for calls of many rows) --------------------------------------------

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
        const int k = 32 * h + 16 * s + 8 * (f >> 1) + 2 * tig;
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
constexpr int kFewRing = 3;     // stages of a warp's ring
// k64 blocks of a stage: four records
template <int MATS> constexpr int kRingBlocks = 4 / MATS;

// 16 + the zero points of the two columns (24 without): as the nibbles, a zero point at the top of
// the mantissa of a number in [16, 32).
template <bool kZeros>
__device__ __forceinline__ void zero_points(const char* record, int per, int h, int gid, float& z0,
                                            float& z1) {
  uint32_t z = 0x0808u;
  if (kZeros) z = *reinterpret_cast<const uint16_t*>(record + 512 + 32 * per + 16 * h + 2 * gid);
  z0 = __uint_as_float(0x41800000u | ((z & 15u) << 19));
  z1 = __uint_as_float(0x41800000u | ((z & 0x0f00u) << 11));
}

// NB k64 blocks of at most 8 rows, in one group (two with kG = 32): fin += the products of MATS
// records a block with the activations xv (two registers per k16 step).  With the weights as
// 16 + q the sum of the activations is needed as well; the tensor cores, which have the time,
// make it.
template <typename T, int MATS, int kG, bool kZeros, int NB>
__device__ __forceinline__ void few_blocks(const char* stage, int matrix_bytes, int rec, int lane,
                                           const uint32_t (&xv)[2][4][2], int first,
                                           float (&fin)[MATS][4]) {
  using T2 = typename Pair<T>::type;
  constexpr int kPer = kG == 32 ? 2 : 1;
  constexpr uint32_t one = Nib<T>::kOne;
  const int gid = lane >> 2;
  // an accumulator's MMAs wait for one another, those of different ones do not: step by step, the
  // sums of the activations and the matrices in turn
  float xs[kPer][4], acc[MATS][kPer][4];
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    uint4 wq[MATS];
#pragma unroll
    for (int m = 0; m < MATS; ++m)
      wq[m] = *(reinterpret_cast<const uint4*>(stage + m * matrix_bytes + b * rec) + lane);
#pragma unroll
    for (int s = 0; s < 4; ++s) {
      const uint32_t(&x)[2] = xv[first + b][s];
      const int h = (s >> 1) & (kPer - 1);
      const bool zero = b == 0 && (s == 0 || (kPer == 2 && s == 2));
      if (zero) mma16816_zero<T>(xs[h], one, one, one, one, x[0], x[1]);
      else mma16816<T>(xs[h], one, one, one, one, x[0], x[1]);
#pragma unroll
      for (int m = 0; m < MATS; ++m) {
        const uint32_t word = s == 0 ? wq[m].x : s == 1 ? wq[m].y : s == 2 ? wq[m].z : wq[m].w;
        const uint32_t a0 = nib_pair<T>(word, 0), a1 = nib_pair<T>(word, 1),
                       a2 = nib_pair<T>(word, 2), a3 = nib_pair<T>(word, 3);
        if (zero) mma16816_zero<T>(acc[m][h], a0, a1, a2, a3, x[0], x[1]);
        else mma16816<T>(acc[m][h], a0, a1, a2, a3, x[0], x[1]);
      }
    }
  }
#pragma unroll
  for (int m = 0; m < MATS; ++m) {
    const char* record = stage + m * matrix_bytes;
#pragma unroll
    for (int h = 0; h < kPer; ++h) {
      float z0, z1;
      zero_points<kZeros>(record, kPer, h, gid, z0, z1);
      const T2 sc = *(reinterpret_cast<const T2*>(record + 512 + 32 * h) + gid);
      const float s0 = Elem<T>::to_f(sc.x), s1 = Elem<T>::to_f(sc.y);
      fin[m][0] += s0 * (acc[m][h][0] - z0 * xs[h][0]);
      fin[m][1] += s0 * (acc[m][h][1] - z0 * xs[h][1]);
      fin[m][2] += s1 * (acc[m][h][2] - z1 * xs[h][0]);
      fin[m][3] += s1 * (acc[m][h][3] - z1 * xs[h][1]);
    }
  }
}

// The `blocks` blocks of a warp's slice (of `per` that the ring holds places for): the activations
// of two blocks are under way while the two before are worked on.  With groups of 128 a slice
// starts on one, and two blocks share their scales.
template <typename T, int MATS, int kG, bool kZeros, typename Issue>
__device__ __forceinline__ void few_slice(WeightRing<MATS, kFewRing>& w, const T* xr, int per,
                                          int blocks, int rec, int lane, float (&fin)[MATS][4],
                                          Issue& issue) {
  uint32_t xn[2][4][2];
  auto load_x = [&](int b) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (b + i < blocks) {
#pragma unroll
        for (int s = 0; s < 8; ++s)
          xn[i][s >> 1][s & 1] = *reinterpret_cast<const uint32_t*>(xr + 64 * (b + i) + 8 * s);
      }
  };
  load_x(0);
  for (int r = 0; r < per; r += kRingBlocks<MATS>) {
    const char* stage = w.wait();
#pragma unroll
    for (int b = 0; b < kRingBlocks<MATS>; b += 2) {
      if (r + b >= blocks) break;
      uint32_t xv[2][4][2];
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int s = 0; s < 8; ++s) xv[i][s >> 1][s & 1] = xn[i][s >> 1][s & 1];
      load_x(r + b + 2);
      const char* from = stage + b * rec;
      if (kG == 128) {
        few_blocks<T, MATS, kG, kZeros, 2>(from, w.matrix_bytes, rec, lane, xv, 0, fin);
      } else {
        few_blocks<T, MATS, kG, kZeros, 1>(from, w.matrix_bytes, rec, lane, xv, 0, fin);
        if (r + b + 1 < blocks)
          few_blocks<T, MATS, kG, kZeros, 1>(from + rec, w.matrix_bytes, rec, lane, xv, 1, fin);
      }
    }
    w.release();
    issue();
  }
}

// Blocks of each of `pieces` slices of K: an even number with groups of 128.
template <int kG> __host__ __device__ __forceinline__ int slice_blocks(int kb, int pieces) {
  const int n = (kb + pieces - 1) / pieces;
  return kG == 128 ? (n + 1) & ~1 : n;
}

constexpr int kFewPitch = 20;  // floats of a row of 16 partial sums

__device__ __forceinline__ void store_partial(float* to, int lane, const float (&fin)[4]) {
  const int gid = lane >> 2, tig = lane & 3;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    to[(2 * tig + (i & 1)) * kFewPitch + gid + 8 * (i >> 1)] = fin[i];
}

template <int kCount, int kSlots>
__device__ __forceinline__ void init_rings(uint64_t (&bar)[kCount][kSlots], int* abort_flag) {
  if ((threadIdx.x & 31) == 0)
    for (int i = 0; i < kSlots; ++i) mbar_init(smem_addr(&bar[threadIdx.x >> 5][i]), 1);
  if (threadIdx.x == 0) *abort_flag = 0;
  fence_barrier_init();
  __syncthreads();
}

// Calls of at most kTableLimit rows need no route preparation: every CTA sorts the rows by expert
// itself (stable, as the route preparation does), in tables for kTableRows.  Up to the limit the
// kernels with a table win, by one measurement on each side of it: 48 rows of 128 experts (2048 x
// 768) take 42 us against 49, 64 rows of 8 experts (4096 x 1536) 58 against 46.
constexpr int kTableLimit = 48;
constexpr int kTableRows = 64;
static_assert(kTableLimit <= kTableRows, "rows of the table");
struct RowTable {
  int row[kTableRows];               // flat row t*k + j of each sorted position
  int place[kTableRows];             // sorted position of each flat row, -1: id >= E
  int chunk_of[kTableRows];          // chunk of each sorted position
  int first[kTableRows + 1];         // first position of each chunk of at most 8 rows
  int expert[kTableRows];            // expert of each chunk
  float weight[kTableRows];          // of each flat row
  int chunks;
  uint32_t id[kTableRows];           // scratch
  unsigned starts[kTableRows / 32];  // scratch

  __device__ __forceinline__ void build(const uint32_t* __restrict__ idx,
                                        const float* __restrict__ weights, int n, int E) {
    const int i = threadIdx.x;
    uint32_t e = 0xffffffffu;
    if (i < kTableRows) {
      if (i < n) {
        e = __ldg(idx + i);
        weight[i] = __ldg(weights + i);
      }
      if (e >= static_cast<uint32_t>(E)) e = 0xffffffffu;
      id[i] = e;
    }
    __syncthreads();
    int before = 0, same = 0, valid = 0;
    if (i < kTableRows) {
      for (int j = 0; j < n; ++j) {
        const uint32_t o = id[j];
        before += o < e || (o == e && j < i);
        same += o == e && j < i;
        valid += o != 0xffffffffu;
      }
      place[i] = e != 0xffffffffu ? before : -1;
      if (e != 0xffffffffu) {
        row[before] = i;
        chunk_of[before] = same % 8 == 0;  // a chunk starts here
      } else if (before < kTableRows) {
        // positions past the valid rows (invalid ids sort last, in order)
        if (i < n) chunk_of[before] = 0;
      }
      if (i >= n) chunk_of[i] = 0;
    }
    __syncthreads();
    bool start = false;
    if (i < kTableRows) {
      start = chunk_of[i] != 0 && i < valid;
      const unsigned b = __ballot_sync(0xffffffffu, start);
      if ((i & 31) == 0) starts[i >> 5] = b;
    }
    __syncthreads();
    if (i < kTableRows) {
      const unsigned upto = starts[i >> 5] & (0xffffffffu >> (31 - (i & 31)));
      const int c = __popc(upto) + (i >= 32 ? __popc(starts[0]) : 0) - 1;
      chunk_of[i] = c;
      if (start) {
        first[c] = i;
        expert[c] = static_cast<int>(id[row[i]]);
      }
      if (i == 0) {
        chunks = __popc(starts[0]) + __popc(starts[1]);
        first[chunks] = valid;
      }
    }
    __syncthreads();
  }
};

// The first product of such a call, in chunks of at most 8 rows.  A unit is (chunk, WN strips of 16
// output columns); the CTA's warps are WN strips x WK pieces of K, so that one token's experts
// spread over the GPU, and nothing but the sum of a unit's WK partial results makes a warp wait
// for another.  The activations come straight from L1 / L2, two blocks ahead.  Rows past the
// chunk's repeat its last one (columns of the product do not mix).  MATS = 2: gate and up.
template <typename T, int MATS, int kG, bool kZeros>
__global__ void __launch_bounds__(kWarps * 32, 3) int4_few_kernel(Int4Params p) {
  constexpr int kSlots = kFewRing;
  constexpr int kBlocks = kRingBlocks<MATS>;
  extern __shared__ __align__(128) char smem[];
  __shared__ alignas(8) uint64_t s_bar[kWarps][kSlots];
  __shared__ int s_abort;
  __shared__ RowTable table;
  float* red = reinterpret_cast<float*>(smem);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int wk = warp % p.wk, wn = warp / p.wk, wn_count = kWarps / p.wk;
  const int kb = p.K / 64, ntiles = p.N / 16, per = slice_blocks<kG>(kb, p.wk);
  const int b0 = min(wk * per, kb), b1 = min(wk * per + per, kb);
  init_rings(s_bar, &s_abort);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  table.build(p.idx, p.sorted_w, p.rows, p.E);
  const int nunits = (ntiles + wn_count - 1) / wn_count;
  const int units = table.chunks * nunits;
  const int matrix_bytes = kBlocks * p.rec;
  WeightRing<MATS, kSlots> w{
      smem + kWarps * MATS * 8 * kFewPitch * 4 + warp * kSlots * MATS * matrix_bytes,
      smem_addr(&s_bar[warp][0]), &s_abort, p.err, lane, matrix_bytes};
  int pu = blockIdx.x, pb = 0;  // the next stage to ask for: unit, first block within [0, per)
  int64_t offset = 0;           // of its first record
  auto locate = [&]() {
    if (pu < units) {
      const int c = pu / nunits;
      // a strip past the last one repeats it, and its results are dropped
      const int nt = min((pu - c * nunits) * wn_count + wn, ntiles - 1);
      offset = ((static_cast<int64_t>(table.expert[c]) * ntiles + nt) * kb + b0) * p.rec;
    }
  };
  auto issue = [&]() {
    if (pu >= units) return;
    w.issue(static_cast<const char*>(p.w[0]) + offset, static_cast<const char*>(p.w[1]) + offset,
            max(min(kBlocks, b1 - b0 - pb), 0) * p.rec);
    offset += matrix_bytes;
    pb += kBlocks;
    if (pb >= per) {
      pb = 0;
      pu += gridDim.x;
      locate();
    }
  };
  locate();
#pragma unroll
  for (int i = 0; i < kSlots - 1; ++i) issue();

  for (int u = blockIdx.x; u < units; u += gridDim.x) {
    const int c = u / nunits;
    const int row0 = table.first[c], rows = table.first[c + 1] - row0;
    const T* xr = static_cast<const T*>(p.x) + 2 * tig + 64 * b0 +
                  static_cast<int64_t>(table.row[row0 + min(gid, rows - 1)] / p.k) * p.K;
    float fin[MATS][4] = {};
    few_slice<T, MATS, kG, kZeros>(w, xr, per, b1 - b0, p.rec, lane, fin, issue);
#pragma unroll
    for (int m = 0; m < MATS; ++m)
      store_partial(red + (warp * MATS + m) * 8 * kFewPitch, lane, fin[m]);
    __syncthreads();
    for (int i = threadIdx.x; i < wn_count * rows * 16; i += kWarps * 32) {
      const int n = i & 15, at = (i >> 4) % rows, strip = (i >> 4) / rows;
      const int col = ((u - c * nunits) * wn_count + strip) * 16 + n;
      if (col >= p.N) continue;
      float v = 0.f, v1 = 0.f;
      for (int q = 0; q < p.wk; ++q) {  // in the order of k
        const float* from = red + ((strip * p.wk + q) * MATS * 8 + at) * kFewPitch + n;
        v += from[0];
        if (MATS == 2) v1 += from[8 * kFewPitch];
      }
      v = act_apply(v, p.act);
      if (MATS == 2) v *= v1;
      // the intermediate is rounded to the 16-bit type that the second product reads
      static_cast<T*>(p.out)[static_cast<int64_t>(row0 + at) * p.N + col] = Elem<T>::from_f(v);
    }
    __syncthreads();
  }
  w.drain();
}

// The second product of a call of at most kTableLimit rows, with the combine: a CTA takes a strip of
// 16 output columns of every token.  A warp's task is (chunk, piece of K); the partial results
// of all tasks meet in shared memory, where the strip's outputs are summed in slot order.
template <typename T, int kG, bool kZeros, int kDownWarps>
__global__ void __launch_bounds__(kDownWarps * 32, 16 / kDownWarps) int4_few_down_kernel(Int4Params p) {
  extern __shared__ __align__(128) char smem[];
  __shared__ alignas(8) uint64_t s_bar[kDownWarps][kFewRing];
  __shared__ int s_abort;
  __shared__ RowTable table;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int gid = lane >> 2, tig = lane & 3;
  const int kb = p.K / 64, ntiles = p.N / 16;
  init_rings(s_bar, &s_abort);
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  table.build(p.idx, p.sorted_w, p.rows, p.E);
  const int chunks = table.chunks;
  // pieces of K: enough tasks for the warps, of three blocks or more
  int pieces = 1;
  while (pieces * 2 * chunks <= kDownWarps && kb >= 6 * pieces) pieces *= 2;
  const int tasks = chunks * pieces, per = slice_blocks<kG>(kb, pieces);
  const int matrix_bytes = kRingBlocks<1> * p.rec;
  float* part = reinterpret_cast<float*>(smem + kDownWarps * kFewRing * matrix_bytes);
  WeightRing<1, kFewRing> w{smem + warp * kFewRing * matrix_bytes, smem_addr(&s_bar[warp][0]),
                            &s_abort, p.err, lane, matrix_bytes};
  int pn = blockIdx.x, pt = warp, pb = 0;  // the next stage to ask for: strip, task, block
  int64_t offset = 0;
  int left = 0;
  auto locate = [&]() {
    if (pt >= tasks) {
      pt = warp;
      pn += gridDim.x;
    }
    if (pn < ntiles && pt < tasks) {
      const int b0 = pt % pieces * per;
      left = min(per, kb - b0);
      offset = ((static_cast<int64_t>(table.expert[pt / pieces]) * ntiles + pn) * kb + b0) * p.rec;
    }
  };
  auto issue = [&]() {
    if (pn >= ntiles || warp >= tasks) return;
    w.issue(static_cast<const char*>(p.w[0]) + offset, nullptr,
            max(min(kRingBlocks<1>, left - pb), 0) * p.rec);
    offset += matrix_bytes;
    pb += kRingBlocks<1>;
    if (pb >= per) {
      pb = 0;
      pt += kDownWarps;
      locate();
    }
  };
  locate();
#pragma unroll
  for (int i = 0; i < kFewRing - 1; ++i) issue();

  for (int nt = blockIdx.x; nt < ntiles; nt += gridDim.x) {
    for (int t = warp; t < tasks; t += kDownWarps) {
      const int c = t / pieces, b0 = t % pieces * per, blocks = min(per, kb - b0);
      const int row0 = table.first[c], rows = table.first[c + 1] - row0;
      const T* xr = static_cast<const T*>(p.x) + 2 * tig + 64 * b0 +
                    static_cast<int64_t>(row0 + min(gid, rows - 1)) * p.K;
      float fin[1][4] = {};
      few_slice<T, 1, kG, kZeros>(w, xr, per, blocks, p.rec, lane, fin, issue);
      store_partial(part + t * 8 * kFewPitch, lane, fin[0]);
    }
    __syncthreads();
    for (int i = threadIdx.x; i < p.rows / p.k * 16; i += kDownWarps * 32) {
      const int n = i & 15, t = i >> 4;
      float v = 0.f;
      for (int j = 0; j < p.k; ++j) {
        const int at = table.place[t * p.k + j];
        if (at < 0) continue;
        const int c = table.chunk_of[at];
        const float* from = part + (c * pieces * 8 + at - table.first[c]) * kFewPitch + n;
        float y = 0.f;
        for (int q = 0; q < pieces; ++q) y += from[q * 8 * kFewPitch];
        v += y * table.weight[t * p.k + j];
      }
      static_cast<T*>(p.out)[static_cast<int64_t>(t) * p.N + nt * 16 + n] = Elem<T>::from_f(v);
    }
    __syncthreads();
  }
  w.drain();
}

// out[t] = sum over the token's slots in slot order, one rounding; four columns a thread.  Bound by
// the slots it reads.
template <typename T>
__global__ void __launch_bounds__(256)
    int4_combine_kernel(const float* __restrict__ slots, const uint32_t* __restrict__ idx, int64_t T_,
                        int k, int H, int E, T* __restrict__ out) {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  const int h4 = H / 4;
  const int64_t total = T_ * h4;
  for (int64_t i = static_cast<int64_t>(blockIdx.x) * blockDim.x + threadIdx.x; i < total;
       i += static_cast<int64_t>(gridDim.x) * blockDim.x) {
    const int64_t t = i / h4;
    const int h = static_cast<int>(i - t * h4) * 4;
    float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int j = 0; j < k; ++j)
      if (__ldg(idx + t * k + j) < static_cast<uint32_t>(E)) {
        const float4 y = __ldcs(reinterpret_cast<const float4*>(slots + (t * k + j) * H + h));
        v.x += y.x;
        v.y += y.y;
        v.z += y.z;
        v.w += y.w;
      }
    *reinterpret_cast<uint2*>(out + t * H + h) = make_uint2(pack2<T>(v.x, v.y), pack2<T>(v.z, v.w));
  }
}

// ---- rows by expert ------------------------------------------------------------------------------

// What the route preparation computes (route_prep.cu: a stable counting sort of the rows by expert,
// offsets and chunk prefix), in one CTA and three barriers: every warp ranks a run of rows of
// its own against a table of counts per warp and expert, the table is summed over the warps, and
// the rows go to base + warps before + rank.  The general kernel takes a barrier for every 512
// rows (4096 rows: 15 us against 5).
constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kSortPer = 4;  // rows of a lane

__device__ __forceinline__ int warp_scan(int v) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int n = __shfl_up_sync(0xffffffffu, v, o);
    if (lane >= o) v += n;
  }
  return v;
}

__global__ void __launch_bounds__(kSortThreads, 1)
    int4_sort_kernel(const uint32_t* __restrict__ idx, const float* __restrict__ weights, int rows,
                     int k, int E, int chunk, int32_t* __restrict__ offsets,
                     int32_t* __restrict__ chunk_prefix, int32_t* __restrict__ sorted_token,
                     float* __restrict__ sorted_w, int32_t* __restrict__ sorted_flat) {
  extern __shared__ int smem_i[];
  int* base = smem_i;                                        // [E]
  uint16_t* counts = reinterpret_cast<uint16_t*>(base + E);  // [kSortWarps][E], then rows before
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  for (int i = threadIdx.x; i < kSortWarps * E / 2; i += kSortThreads)
    reinterpret_cast<uint32_t*>(counts)[i] = 0u;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  uint32_t e[kSortPer];
  float w[kSortPer];
  int rank[kSortPer];
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const int r = warp * 32 * kSortPer + i * 32 + lane;
    e[i] = r < rows ? __ldg(idx + r) : 0xffffffffu;
    w[i] = r < rows ? __ldg(weights + r) : 0.f;
  }
  __syncthreads();
  uint16_t* mine = counts + warp * E;
#pragma unroll
  for (int i = 0; i < kSortPer; ++i) {
    const bool in = e[i] < static_cast<uint32_t>(E);
    const unsigned peers = __match_any_sync(0xffffffffu, in ? e[i] : 0xffffffffu);
    const int before = __popc(peers & ((1u << lane) - 1u));
    if (in) rank[i] = mine[e[i]] + before;
    __syncwarp();
    if (in && before == 0) mine[e[i]] = static_cast<uint16_t>(mine[e[i]] + __popc(peers));
    __syncwarp();
  }
  __syncthreads();
  for (int x = threadIdx.x; x < E; x += kSortThreads) {
    int run = 0;
#pragma unroll 8
    for (int v = 0; v < kSortWarps; ++v) {
      const int c = counts[v * E + x];
      counts[v * E + x] = static_cast<uint16_t>(run);
      run += c;
    }
    base[x] = run;
  }
  __syncthreads();
  if (warp == 0) {
    int rows_before = 0, chunks_before = 0, most = 0;
    for (int x0 = 0; x0 < E; x0 += 32) {
      const int x = x0 + lane;
      const int c = x < E ? base[x] : 0, n = (c + chunk - 1) / chunk;
      const int ic = warp_scan(c), in = warp_scan(n);
      if (x < E) {
        base[x] = rows_before + ic - c;
        offsets[x] = rows_before + ic - c;
        chunk_prefix[x] = chunks_before + in - n;
      }
      most = max(most, static_cast<int>(__reduce_max_sync(0xffffffffu, static_cast<unsigned>(c))));
      rows_before += __shfl_sync(0xffffffffu, ic, 31);
      chunks_before += __shfl_sync(0xffffffffu, in, 31);
    }
    if (lane == 0) {
      offsets[E] = rows_before;
      offsets[E + 1] = most;
      chunk_prefix[E] = chunks_before;
    }
  }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < kSortPer; ++i)
    if (e[i] < static_cast<uint32_t>(E)) {
      const int r = warp * 32 * kSortPer + i * 32 + lane;
      const int at = base[e[i]] + mine[e[i]] + rank[i];
      sorted_token[at] = r / k;
      sorted_w[at] = w[i];
      sorted_flat[at] = r;
    }
}

int grid_for(int64_t n, int num_sms) {
  const int64_t b = (n + 255) / 256, cap = static_cast<int64_t>(num_sms) * 16;
  return static_cast<int>(b < cap ? b : cap);
}

template <typename T, int MATS, int kG, bool kZeros>
struct Few {
  static constexpr auto kernel = int4_few_kernel<T, MATS, kG, kZeros>;
  static size_t smem(int rec) {
    return static_cast<size_t>(kWarps) * MATS *
           (8 * kFewPitch * 4 + kFewRing * kRingBlocks<MATS> * rec);
  }
  static bool launch(Int4Params p, int num_sms, cudaStream_t s) {
    // pieces of K: there are few units, so as many as leave a warp three blocks
    p.wk = kWarps;
    while (p.wk > 1 && p.K / 64 < 3 * p.wk) p.wk /= 2;
    // three CTAs on an SM: 3 x (10 + 52 + 3 KB) with groups of 64 and more
    return launch_dependent(kernel, num_sms * 3, kWarps * 32, smem(p.rec), s, p);
  }
};

// kDownWarps 16: one CTA on an SM, for at most as many strips as SMs; 8: two.
template <typename T, int kG, bool kZeros, int kDownWarps>
struct FewDown {
  static constexpr auto kernel = int4_few_down_kernel<T, kG, kZeros, kDownWarps>;
  static size_t smem(int rec) { return smem(rec, kTableRows); }
  // partial results: one task per chunk, or at most kDownWarps with K in pieces
  static size_t smem(int rec, int rows) {
    const int tasks = rows > kDownWarps ? rows : kDownWarps;
    return static_cast<size_t>(kDownWarps) * kFewRing * kRingBlocks<1> * rec +
           static_cast<size_t>(tasks) * 8 * kFewPitch * 4;
  }
  static bool launch(const Int4Params& p, int num_sms, cudaStream_t s) {
    const int most = num_sms * (16 / kDownWarps);
    const int grid = p.N / 16 < most ? p.N / 16 : most;
    return launch_dependent(kernel, grid, kDownWarps * 32, smem(p.rec, p.rows), s, p);
  }
};

template <typename K> bool allow_smem() {
  return cudaFuncSetAttribute(K::kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(K::smem(kMaxRecord))) == cudaSuccess;
}
template <typename T, int kG, bool kZeros> bool few_attributes() {
  return allow_smem<Few<T, 2, kG, kZeros>>() && allow_smem<Few<T, 1, kG, kZeros>>() &&
         allow_smem<FewDown<T, kG, kZeros, 8>>() && allow_smem<FewDown<T, kG, kZeros, 16>>();
}
template <typename T> bool few_attributes() {
  return few_attributes<T, 32, false>() && few_attributes<T, 32, true>() &&
         few_attributes<T, 64, false>() && few_attributes<T, 64, true>() &&
         few_attributes<T, 128, false>() && few_attributes<T, 128, true>();
}

template <typename T, int kG, bool kZeros>
bool launch_table(const Int4Params& g1, const Int4Params& g2, int num_sms,
                  cudaEvent_t between, cudaStream_t s) {
  const bool ok = g1.w[1] ? Few<T, 2, kG, kZeros>::launch(g1, num_sms, s)
                          : Few<T, 1, kG, kZeros>::launch(g1, num_sms, s);
  if (between) cudaEventRecord(between, s);
  return ok &&
         (g2.N / 16 <= num_sms ? FewDown<T, kG, kZeros, 16>::launch(g2, num_sms, s)
                               : FewDown<T, kG, kZeros, 8>::launch(g2, num_sms, s));
}
template <typename T, int kG>
bool launch_table(const Int4Params& g1, const Int4Params& g2, int num_sms,
                  cudaEvent_t between, cudaStream_t s) {
  return g1.zeros ? launch_table<T, kG, true>(g1, g2, num_sms, between, s)
                  : launch_table<T, kG, false>(g1, g2, num_sms, between, s);
}
template <typename T>
bool launch_table(const Int4Params& g1, const Int4Params& g2, int num_sms,
                  cudaEvent_t between, cudaStream_t s) {
  return g1.G == 32   ? launch_table<T, 32>(g1, g2, num_sms, between, s)
         : g1.G == 64 ? launch_table<T, 64>(g1, g2, num_sms, between, s)
                      : launch_table<T, 128>(g1, g2, num_sms, between, s);
}

template <typename T>
bool launch_combine(const Int4Params& g2, const uint32_t* idx, int64_t T_, int k, void* out,
                    int num_sms, cudaStream_t s) {
  return launch_dependent(int4_combine_kernel<T>, grid_for(T_ * (g2.N / 4), num_sms), 256, 0, s,
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

bool int4_set_attributes() {
  return few_attributes<__nv_bfloat16>() && few_attributes<__half>() &&
         int4_many_set_attributes() &&
         cudaFuncSetAttribute(int4_sort_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize,
                              route_prep_max_experts() * (4 + 2 * kSortWarps)) == cudaSuccess;
}

void launch_int4_expand(int dtype, const void* w, int E, int K, int N, int G, bool zeros,
                        bool trans, void* out, cudaStream_t s) {
  if (dtype == kBF16) expand<__nv_bfloat16>(w, E, K, N, G, zeros, trans, out, s);
  else expand<__half>(w, E, K, N, G, zeros, trans, out, s);
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

int int4_table_rows() { return kTableLimit; }

static size_t sort_smem(int E) {
  return sizeof(int) * E + sizeof(uint16_t) * kSortWarps * static_cast<size_t>(E);
}

bool launch_int4_sort(const uint32_t* idx, const float* weights, int64_t rows, int k, int E,
                      int chunk, int32_t* offsets, int32_t* chunk_prefix, int32_t* sorted_token,
                      float* sorted_w, int32_t* sorted_flat, cudaStream_t s) {
  return launch_dependent(int4_sort_kernel, 1, kSortThreads, sort_smem(E), s, idx, weights,
                          static_cast<int>(rows), k, E, chunk, offsets, chunk_prefix, sorted_token,
                          sorted_w, sorted_flat);
}
int64_t int4_sort_rows() { return kSortThreads * kSortPer; }

int launch_int4_table_ffn(int dtype, const Int4Params& g1, const Int4Params& g2, int num_sms,
                          cudaEvent_t between, cudaStream_t s) {
  const bool ok = dtype == kBF16 ? launch_table<__nv_bfloat16>(g1, g2, num_sms, between, s)
                                 : launch_table<__half>(g1, g2, num_sms, between, s);
  return ok ? 2 : 0;
}

int launch_int4_ffn(int dtype, const Int4Params& g1, const Int4Params& g2, const uint32_t* idx,
                    int64_t num_tokens, int k, void* out, int num_sms, cudaEvent_t after1,
                    cudaEvent_t after2, cudaStream_t s) {
  bool ok = launch_int4_many(dtype, g1, g2, num_sms, after1, s);
  if (after2) cudaEventRecord(after2, s);
  ok = ok && (dtype == kBF16
                  ? launch_combine<__nv_bfloat16>(g2, idx, num_tokens, k, out, num_sms, s)
                  : launch_combine<__half>(g2, idx, num_tokens, k, out, num_sms, s));
  return ok ? 3 : 0;
}

}  // namespace cmoe
