// Q, many rows per expert: the products on the fifth-generation tensor cores.
//
// A tile is two panels of 128 weight columns (the same columns of gate and up, or 256 columns of one
// matrix) times at most 64 rows of one expert.  The weights are the MMA's 128-row operand and
// come from tensor memory: sixteen warps, a strip of 16 columns each, stream their records
// through rings in shared memory, unpack them in registers -- (q - z) exactly, times the scale,
// one rounding to the 16-bit type, as weights held in that type have -- and store them as they
// lie: the packed fragment order is the 16x128b shape of tcgen05.st, so nothing is shuffled and
// shared memory carries only the packed nibbles.  The rows are the other operand, gathered by
// cp.async into the 128-byte swizzle.  The sums stay in tensor memory for all of K (two sets, so
// that the epilogue of a tile runs under the next one) and leave it one weight column per thread.
//
// What bounds it: issue slots.  A record of 1024 weights takes 60 warp instructions to unpack (for
// a pair of weights a lane under two to place the nibbles, one to subtract, one to scale) and
// 127 with copies, barriers and stores; at the 0.7 instructions a cycle that a scheduler reaches an SM
// unpacks one in 45 cycles, against 24 cycles of its share of the memory rate.  The MMAs take 40
// cycles each at 64 rows or fewer, 20 a record.  512 tokens of 128 experts (2048 x 768, top 8): 82 us
// for gate and up (214 MB), 44 us for down.  What it took to get there: sixteen unpacking warps
// instead of eight, hand-overs of two blocks, an issuer warp whose addresses are uniform (one
// lane alone spent 1500 cycles a block), a warp that feeds all rings, barriers tested ahead.
#include <stdint.h>

#include "common.cuh"
#include "int4.cuh"
#include "kernels.h"

namespace cmoe {

namespace {

constexpr int kTileRows = 64;
constexpr int kUnpackWarps = 16, kOutWarps = 4, kGatherWarps = 4;
constexpr int kThreads = (kUnpackWarps + kOutWarps + kGatherWarps + 2) * 32;
constexpr int kStageBlocks = 2;           // k64 blocks that are handed over at once
constexpr int kStages = 2;                // of weights in tensor memory
constexpr int kXSlots = 4;                // stages of rows in shared memory
constexpr int kXBytes = kTileRows * 128;  // a block's rows
constexpr int kRingSlots = 3, kRingBlocks = 4;
constexpr int kAccCols = 2 * kTileRows;   // of one set of sums, two panels
constexpr int kACols = 2 * 32;            // of one block of weights
constexpr int kTmemCols = 512;
static_assert(2 * kAccCols + kStages * kStageBlocks * kACols <= kTmemCols, "tensor memory");

// D[tmem] (+)= A[tmem] * B[smem], kind::f16.
__device__ __forceinline__ void umma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t b_desc,
                                            uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(b_desc), "r"(idesc), "r"(accumulate)
      : "memory");
}

// 16 lanes x 32 columns: register 2 j + r of lane (gid, tig) goes to lane gid + 8 r, column 4 j + tig.
__device__ __forceinline__ void tmem_st_16x128b_x8(uint32_t taddr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.16x128b.x8.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st_wait() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}

template <typename T> struct Fmt;
template <> struct Fmt<__half> { static constexpr uint32_t v = 0; };
template <> struct Fmt<__nv_bfloat16> { static constexpr uint32_t v = 1; };

// The 16-bit pattern of 16 + z, twice.
template <typename T> __device__ __forceinline__ uint32_t zero_pair(uint32_t z) {
  return Nib<T>::kMagic | ((z << Nib<T>::kShift) * 0x10001u);
}

// A group's scales and zero points (as 16 + z) of a lane's two columns.
template <typename T> struct Group {
  typename Pair<T>::type scale[2], off[2];
};
template <typename T, bool kZeros>
__device__ __forceinline__ void load_group(const char* record, int per, int h, int lane,
                                           Group<T>& g) {
  using T2 = typename Pair<T>::type;
  const int gid = lane >> 2;
  const T2 s = *(reinterpret_cast<const T2*>(record + 512 + 32 * h) + gid);
  g.scale[0].x = g.scale[0].y = s.x;
  g.scale[1].x = g.scale[1].y = s.y;
  uint32_t z = 0x0808u;
  if (kZeros) z = *reinterpret_cast<const uint16_t*>(record + 512 + 32 * per + 16 * h + 2 * gid);
  const uint32_t z0 = zero_pair<T>(z & 15u), z1 = zero_pair<T>((z >> 8) & 15u);
  g.off[0] = *reinterpret_cast<const T2*>(&z0);
  g.off[1] = *reinterpret_cast<const T2*>(&z1);
}

// The record's weights in the order of tmem_st_16x128b_x8; `g` holds its first group.
template <typename T, bool kZeros>
__device__ __forceinline__ void unpack_record(const char* record, int per, int lane, Group<T>& g,
                                              uint32_t (&out)[16]) {
  using T2 = typename Pair<T>::type;
  const uint4 wq = *(reinterpret_cast<const uint4*>(record) + lane);
  const uint32_t word[4] = {wq.x, wq.y, wq.z, wq.w};
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    if (h == 1 && per == 2) load_group<T, kZeros>(record, per, 1, lane, g);
#pragma unroll
    for (int c = 0; c < 4; ++c)
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        const uint32_t u = nib_pair<T>(word[2 * h + (c >> 1)], 2 * (c & 1) + r);
        const T2 v = __hmul2(__hsub2(*reinterpret_cast<const T2*>(&u), g.off[r]), g.scale[r]);
        out[2 * (4 * h + c) + r] = *reinterpret_cast<const uint32_t*>(&v);
      }
  }
}

// kDual: the panels are gate and up, else the two halves of 256 columns.
template <typename T, bool kDual, bool kDown, bool kZeros>
__global__ void __launch_bounds__(kThreads, 1) int4_many_kernel(Int4Params p) {
  constexpr int kCols = kDual ? 128 : 256;  // output columns of a unit
  extern __shared__ __align__(128) char smem_raw[];
  __shared__ alignas(8) uint64_t s_ring[kUnpackWarps][kRingSlots], s_free[kUnpackWarps][kRingSlots];
  __shared__ alignas(8) uint64_t s_full[kStages], s_empty[kStages];
  __shared__ alignas(8) uint64_t acc_full[2], acc_empty[2], s_done;
  __shared__ uint32_t s_tmem;
  __shared__ int s_abort, s_never;
  const uint32_t raw = smem_addr(smem_raw);
  const uint32_t x_base = (raw + 1023u) & ~1023u;
  char* x_smem = smem_raw + (x_base - raw);
  char* rings = x_smem + kXSlots * kStageBlocks * kXBytes;
  int32_t* s_cp = reinterpret_cast<int32_t*>(rings + kUnpackWarps * kRingSlots * kRingBlocks * p.rec);
  int32_t* s_off = s_cp + p.E + 1;
  // from a shuffle, so that the compiler knows it to be the same in the warp
  const int warp = __shfl_sync(0xffffffffu, static_cast<int>(threadIdx.x >> 5), 0);
  const int lane = threadIdx.x & 31;
  const int E = p.E, kb = p.K / 64, MT = (p.N + kCols - 1) / kCols;

  if (threadIdx.x == 0) {
    for (int w = 0; w < kUnpackWarps; ++w)
      for (int i = 0; i < kRingSlots; ++i) {
        mbar_init(smem_addr(&s_ring[w][i]), 1);
        mbar_init(smem_addr(&s_free[w][i]), 1);
      }
    for (int i = 0; i < kStages; ++i) {
      mbar_init(smem_addr(&s_full[i]), kUnpackWarps + kGatherWarps);
      mbar_init(smem_addr(&s_empty[i]), 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(smem_addr(&acc_full[i]), 1);
      mbar_init(smem_addr(&acc_empty[i]), kOutWarps);
    }
    mbar_init(smem_addr(&s_done), 1);
    s_abort = s_never = 0;
    fence_barrier_init();
  }
  if (warp == kThreads / 32 - 1) {
    tmem_alloc(smem_addr(&s_tmem), kTmemCols);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem, tmem_a = tmem + 2 * kAccCols;
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  for (int i = threadIdx.x; i <= E; i += kThreads) {
    s_cp[i] = __ldg(p.chunk_prefix + i);
    s_off[i] = __ldg(p.offsets + i);
  }
  __syncthreads();
  const int64_t units = static_cast<int64_t>(s_cp[E]) * MT;
  struct Unit {
    int e, mt, row0, rows;
  };
  auto unit_of = [&](int64_t u) {
    Unit d;
    const int c = static_cast<int>(u / MT);
    d.mt = static_cast<int>(u % MT);
    d.e = expert_of_tile_smem(s_cp, E, c);
    d.row0 = s_off[d.e] + (c - s_cp[d.e]) * kTileRows;
    d.rows = min(kTileRows, s_off[d.e + 1] - d.row0);
    return d;
  };

  if (warp < kUnpackWarps) {
    // ------------------------------------------------------------------ weights into TMEM
    const int panel = warp >> 3;
    const int strip = 2 * (warp & 3) + ((warp >> 2) & 1);  // in this warp's quarter of the lanes
    const uint32_t lanes = static_cast<uint32_t>(16 * strip) << 16;
    const int per = p.G == 32 ? 2 : 1;
    const int matrix_bytes = kRingBlocks * p.rec;
    WeightRing<1, kRingSlots> w{rings + warp * kRingSlots * matrix_bytes,
                                      smem_addr(&s_ring[warp][0]), &s_abort, p.err, lane,
                                      matrix_bytes};
    int at = 0;
    uint32_t phase = 0, landed = 0;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
      for (int r = 0; r < kb; r += kRingBlocks) {
        if (!landed) w.wait();
        const char* stage = w.stage();
#pragma unroll
        for (int b = 0; b < kRingBlocks; b += kStageBlocks) {
          if (r + b >= kb) break;
          const uint32_t empty = smem_addr(&s_empty[at]);
          const uint32_t free_now = mbar_test(empty, phase ^ 1u);
          const uint32_t to = tmem_a + at * kStageBlocks * kACols + panel * 32 + lanes;
          Group<T> g;
#pragma unroll
          for (int i = 0; i < kStageBlocks; ++i) {
            if (r + b + i >= kb) break;
            const char* record = stage + (b + i) * p.rec;
            // the two blocks of a stage are one group of 128
            if (i == 0 || p.G != 128) load_group<T, kZeros>(record, per, 0, lane, g);
            uint32_t regs[16];
            unpack_record<T, kZeros>(record, per, lane, g, regs);
            if (i == 0) {
              // after a wait that ran out this goes on with what is there, to the end of the units
              if (!free_now)
                mbar_wait_parked(empty, phase ^ 1u, &s_abort, p.err, kErrWaitEmpty);
              __syncwarp();
              tc_fence_after();
            }
            tmem_st_16x128b_x8(to + i * kACols, regs);
          }
          tmem_st_wait();
          tc_fence_before();
          __syncwarp();
          if (lane == 0) mbar_arrive(smem_addr(&s_full[at]));
          at ^= 1;
          phase ^= at == 0;
        }
        const int slot = w.slot;
        w.release();
        landed = w.test();
        if (lane == 0) mbar_arrive(smem_addr(&s_free[warp][slot]));
      }
    }
    w.drain();
  } else if (warp < kUnpackWarps + kOutWarps) {
    // ------------------------------------------------------------------ sums out of TMEM
    const int q = warp & 3;
    int buf = 0;
    uint32_t phase = 0;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
      const Unit d = unit_of(u);
      const int col = d.mt * kCols + 32 * q + lane;
      const bool first = col < p.N, second = col + 128 < p.N;
      const bool ok = mbar_wait_parked(smem_addr(&acc_full[buf]), phase, &s_abort, p.err,
                                        kErrWaitAccFull);
      if (!__all_sync(0xffffffffu, ok)) break;
      tc_fence_after();
      const uint32_t t = tmem + buf * kAccCols + (static_cast<uint32_t>(32 * q) << 16);
      for (int r0 = 0; r0 < d.rows; r0 += 16) {
        uint32_t v[16], g[16];
        tmem_ld_32x32b_x16(t + r0, v);
        tmem_ld_32x32b_x16(t + kTileRows + r0, g);
        int flat = 0;
        float wt = 0.f;
        if (kDown) {  // a lane's row, handed around below
          const int row = d.row0 + min(r0 + (lane & 15), d.rows - 1);
          flat = __ldg(p.sorted_flat + row);
          wt = __ldg(p.sorted_w + row);
        }
        tmem_ld_wait();
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          const int64_t row = kDown ? __shfl_sync(0xffffffffu, flat, i) : d.row0 + r0 + i;
          const float w = kDown ? __shfl_sync(0xffffffffu, wt, i) : 1.f;
          if (r0 + i < d.rows) {
            float y = __uint_as_float(v[i]), y2 = __uint_as_float(g[i]);
            if (kDown) {
              float* out = static_cast<float*>(p.out) + row * p.N + col;
              if (first) out[0] = y * w;
              if (second) out[128] = y2 * w;
            } else {
              // the intermediate is rounded to the 16-bit type that the second product reads
              T* out = static_cast<T*>(p.out) + row * p.N + col;
              y = act_apply(y, p.act);
              if (kDual) y *= y2;
              if (first) out[0] = Elem<T>::from_f(y);
              if (!kDual && second) out[128] = Elem<T>::from_f(act_apply(y2, p.act));
            }
          }
        }
      }
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(smem_addr(&acc_empty[buf]));
      buf ^= 1;
      phase ^= buf == 0;
    }
  } else if (warp < kUnpackWarps + kOutWarps + kGatherWarps) {
    // ------------------------------------------------------------------ rows into shared memory
    // Thread g copies 16-byte piece g % 8 of each block's rows q + 16 i (q = g / 8) to its place in
    // the 128-byte swizzle (piece c of row r at c ^ (r % 8)).  Rows past the tile's repeat its
    // last one; their sums are not read.  The copies run two stages ahead: those of stage
    // n + 2 take the slot of stage n - 2, whose MMAs are done when stage n may be filled.
    const int g = threadIdx.x - (kUnpackWarps + kOutWarps) * 32;
    const int c8 = g & 7, q = g >> 3;
    const uint32_t to = x_base + q * 128 + ((c8 ^ (q & 7)) << 4);
    const T* src[4];
    int64_t lu = blockIdx.x;
    int lb = 0, lrows = 0, slot = 0;
    auto locate = [&]() {
      if (lu >= units) return;
      const Unit d = unit_of(lu);
      lrows = d.rows;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int r = d.row0 + min(q + 16 * i, d.rows - 1);
        src[i] = static_cast<const T*>(p.x) +
                 static_cast<int64_t>(kDown ? r : __ldg(p.sorted_token + r)) * p.K + c8 * 8;
      }
    };
    auto load = [&]() {
      if (lu < units) {
        const uint32_t dst = to + slot * kStageBlocks * kXBytes;
#pragma unroll
        for (int j = 0; j < kStageBlocks; ++j)
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (16 * i < lrows && lb + j < kb)
              cp_async16(dst + j * kXBytes + i * 2048, src[i] + (lb + j) * 64);
        lb += kStageBlocks;
        if (lb >= kb) {
          lb = 0;
          lu += gridDim.x;
          locate();
        }
      }
      asm volatile("cp.async.commit_group;" ::: "memory");
      slot = (slot + 1) & (kXSlots - 1);
    };
    locate();
    load();
    load();
    int at = 0;
    uint32_t phase = 0;
    bool ok = true;
    for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
      for (int b = 0; b < kb; b += kStageBlocks) {
        ok = mbar_wait_parked(smem_addr(&s_empty[at]), phase ^ 1u, &s_abort, p.err, kErrWaitEmpty);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        load();
        asm volatile("cp.async.wait_group 2;" ::: "memory");
        __syncwarp();  // the MMA issuer orders these writes before its reads
        if (lane == 0) mbar_arrive(smem_addr(&s_full[at]));
        at ^= 1;
        phase ^= at == 0;
      }
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
  } else if (warp == kUnpackWarps + kOutWarps + kGatherWarps) {
    // ------------------------------------------------------------------ weight copies
    // Lane w feeds the ring of unpacking warp w, kRingBlocks records at a time.
    if (lane < kUnpackWarps) {
      const int panel = lane >> 3;
      const int strip = 2 * (lane & 3) + ((lane >> 2) & 1);
      const uint32_t full = smem_addr(&s_ring[lane][0]), empty = smem_addr(&s_free[lane][0]);
      const uint32_t stage_bytes = kRingBlocks * p.rec;
      const uint32_t to = smem_addr(rings) + lane * kRingSlots * stage_bytes;
      int slot = 0;
      uint32_t phase = 0;
      bool ok = true;
      for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
        const Unit d = unit_of(u);
        // a strip past the last column repeats the last one; its sums are not read
        const int at = min(d.mt * (kCols / 16) + (kDual ? 0 : panel * 8) + strip, p.N / 16 - 1);
        const char* src = static_cast<const char*>(p.w[kDual ? panel : 0]) +
                          (static_cast<int64_t>(d.e) * (p.N / 16) + at) * kb * p.rec;
        for (int b = 0; b < kb; b += kRingBlocks) {
          ok = mbar_wait_parked(empty + 8 * slot, phase ^ 1u, &s_abort, p.err, kErrWaitEmpty);
          if (!ok) break;
          const uint32_t bytes = min(kRingBlocks, kb - b) * p.rec;
          mbar_arrive_expect_tx(full + 8 * slot, bytes);
          bulk_load(to + slot * stage_bytes, src, bytes, full + 8 * slot);
          src += stage_bytes;
          if (++slot == kRingSlots) {
            slot = 0;
            phase ^= 1u;
          }
        }
      }
    }
  } else {
    // ------------------------------------------------------------------ MMA issuer
    // The whole warp walks the units, so that descriptors and addresses are uniform values; one
    // elected lane issues.  With one lane alone in this branch, two waits and eight MMAs took
    // the issuer 1500 cycles a block among 24 busy warps, and set the pace.
    uint32_t elected;
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b32 r;\n\t"
        "elect.sync r|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(elected));
    int at = 0, slot = 0, buf = 0;
    uint32_t phase = 0, acc_phase = 0;
    bool ok = true;
    const uint64_t desc0 = umma_sdesc(x_base, 16, 1024);
    for (int64_t u = blockIdx.x; ok && u < units; u += gridDim.x) {
      const int rows = unit_of(u).rows;
      const uint32_t idesc = umma_idesc(Fmt<T>::v, 0, 128, (rows + 15) & ~15);
      const uint32_t acc = tmem + buf * kAccCols;
      ok = mbar_wait_parked(smem_addr(&acc_empty[buf]), acc_phase ^ 1u, &s_abort, p.err,
                            kErrWaitAccEmpty);
      if (!__all_sync(0xffffffffu, ok)) break;
      for (int b = 0; b < kb; b += kStageBlocks) {
        ok = mbar_wait_parked(smem_addr(&s_full[at]), phase, &s_abort, p.err, kErrWaitFull);
        ok = __all_sync(0xffffffffu, ok);
        if (!ok) break;
        if (elected) {
          fence_proxy_async_smem();  // the rows were written through the generic proxy
          tc_fence_after();
          const uint64_t desc = desc0 + slot * (kStageBlocks * kXBytes >> 4);
          const uint32_t a = tmem_a + at * kStageBlocks * kACols;
#pragma unroll
          for (int i = 0; i < kStageBlocks; ++i)
            if (b + i < kb) {
#pragma unroll
              for (int ks = 0; ks < 4; ++ks)
#pragma unroll
                for (int m = 0; m < 2; ++m)
                  umma_f16_ts(acc + m * kTileRows, a + i * kACols + m * 32 + ks * 8,
                              desc + i * (kXBytes >> 4) + ks * 2, idesc, b + i + ks > 0);
            }
          umma_commit(smem_addr(&s_empty[at]));
          if (b + kStageBlocks >= kb) umma_commit(smem_addr(&acc_full[buf]));
        }
        __syncwarp();
        at ^= 1;
        phase ^= at == 0;
        slot = (slot + 1) & (kXSlots - 1);
      }
      buf ^= 1;
      acc_phase ^= buf == 0;
    }
    // every MMA is done before the tensor memory and the operands go
    if (elected) umma_commit(smem_addr(&s_done));
    __syncwarp();
    mbar_wait_parked(smem_addr(&s_done), 0, &s_never, p.err, kErrWaitDrain);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == kThreads / 32 - 1) tmem_dealloc(tmem, kTmemCols);
}

size_t smem_bytes(int rec, int E) {
  return 1024 + static_cast<size_t>(kXSlots) * kStageBlocks * kXBytes +
         static_cast<size_t>(kUnpackWarps) * kRingSlots * kRingBlocks * rec +
         static_cast<size_t>(2 * E + 2) * sizeof(int32_t);
}

template <typename T, bool kDual, bool kDown, bool kZeros>
bool attribute() {
  return cudaFuncSetAttribute(int4_many_kernel<T, kDual, kDown, kZeros>,
                              cudaFuncAttributeMaxDynamicSharedMemorySize,
                              static_cast<int>(smem_bytes(kMaxRecord, route_prep_max_experts()))) ==
         cudaSuccess;
}

template <typename T, bool kZeros>
bool launch(const Int4Params& g1, const Int4Params& g2, int num_sms, cudaEvent_t between,
            cudaStream_t s) {
  const size_t smem = smem_bytes(g1.rec, g1.E);
  const bool ok =
      g1.w[1] ? launch_dependent(int4_many_kernel<T, true, false, kZeros>, num_sms, kThreads, smem, s,
                                 g1)
              : launch_dependent(int4_many_kernel<T, false, false, kZeros>, num_sms, kThreads, smem,
                                 s, g1);
  if (between) cudaEventRecord(between, s);
  return ok && launch_dependent(int4_many_kernel<T, false, true, kZeros>, num_sms, kThreads, smem, s,
                                g2);
}

template <typename T, bool kZeros> bool attributes() {
  return attribute<T, true, false, kZeros>() && attribute<T, false, false, kZeros>() &&
         attribute<T, false, true, kZeros>();
}

}  // namespace

int int4_many_rows() { return kTileRows; }

bool int4_many_set_attributes() {
  return attributes<__nv_bfloat16, false>() && attributes<__nv_bfloat16, true>() &&
         attributes<__half, false>() && attributes<__half, true>();
}

bool launch_int4_many(int dtype, const Int4Params& g1, const Int4Params& g2, int num_sms,
                      cudaEvent_t between, cudaStream_t s) {
  if (dtype == kBF16)
    return g1.zeros ? launch<__nv_bfloat16, true>(g1, g2, num_sms, between, s)
                    : launch<__nv_bfloat16, false>(g1, g2, num_sms, between, s);
  return g1.zeros ? launch<__half, true>(g1, g2, num_sms, between, s)
                  : launch<__half, false>(g1, g2, num_sms, between, s);
}

}  // namespace cmoe
