// Pieces shared by the kernels on 4-bit expert weights (moe_int4.cu, moe_int4_mma.cu).
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>

#include "common.cuh"

namespace cmoe {
namespace {

// mbar_wait_bounded that parks the warp in each try (up to 10 us) instead of polling, so that the
// waiting ones of an SM's 26 warps take no issue slots.  (No faster than polling when measured.)
__device__ __forceinline__ bool mbar_wait_parked(uint32_t bar, uint32_t parity,
                                                 volatile int* abort_flag, uint32_t* err,
                                                 uint32_t code) {
  unsigned long long t0 = 0;
  for (;;) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity), "r"(10000u)
        : "memory");
    if (ok) return true;
    if (*abort_flag) return false;
    const unsigned long long now = globaltimer_ns();
    if (t0 == 0) t0 = now;
    if (now - t0 > kWaitLimitNs) {
      *abort_flag = 1;
      if (err) atomicOr(err, code);
      return false;
    }
  }
}

// Whether the phase is complete, without waiting.  The answer takes some hundred cycles on a busy
// SM, so it is asked for ahead of the work before the wait.
__device__ __forceinline__ uint32_t mbar_test(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok;
}

constexpr int kMaxRecord = 608;  // int4_record_bytes(32, true)

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
  // (w & mask) | magic in one instruction, both from registers
  uint32_t r;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;"
      : "=r"(r)
      : "r"(rotr(w, 4 * i)), "r"(Nib<T>::kMask), "r"(Nib<T>::kMagic));
  return r;
}

template <typename T> struct Pair;
template <> struct Pair<__nv_bfloat16> { using type = __nv_bfloat162; };
template <> struct Pair<__half> { using type = __half2; };

__device__ __forceinline__ void bulk_load(uint32_t dst, const void* src, uint32_t bytes,
                                          uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}

// A warp's ring of kSlots stages in shared memory, a stage holding `blocks` records of each of MATS
// matrices.  One lane issues bulk copies that signal a barrier per stage, so a warp waits for no
// other one, and the ring runs ahead across units of work: memory stays busy while a unit is
// finished.
template <int MATS, int kSlots>
struct WeightRing {
  char* ring;
  uint32_t bars;  // kSlots barriers
  volatile int* abort_flag;
  uint32_t* err;
  int lane, matrix_bytes;  // of a stage, per matrix
  int slot_in = 0, slot = 0;
  uint32_t phase = 0;

  __device__ __forceinline__ void issue(const char* src0, const char* src1, uint32_t bytes) {
    if (lane == 0) {
      const uint32_t bar = bars + 8 * slot_in;
      mbar_arrive_expect_tx(bar, MATS * bytes);
      if (bytes) {
        const uint32_t dst = smem_addr(ring) + slot_in * MATS * matrix_bytes;
        bulk_load(dst, src0, bytes, bar);
        if (MATS == 2) bulk_load(dst + matrix_bytes, src1, bytes, bar);
      }
    }
    slot_in = slot_in + 1 == kSlots ? 0 : slot_in + 1;
  }
  // The stage's records, or whatever is there once a wait has run out (the error word is set).
  __device__ __forceinline__ const char* wait() {
    mbar_wait_parked(bars + 8 * slot, phase, abort_flag, err, kErrWaitFull);
    return ring + slot * MATS * matrix_bytes;
  }
  __device__ __forceinline__ uint32_t test() { return mbar_test(bars + 8 * slot, phase); }
  __device__ __forceinline__ const char* stage() const { return ring + slot * MATS * matrix_bytes; }
  // After a wait that ran out: no copy may land once the CTA is gone (each wait again bounded).
  __device__ __forceinline__ void drain() {
    if (!*abort_flag) return;
    const unsigned long long t0 = globaltimer_ns();
    for (int i = 0; i < kSlots; ++i)
      while (!mbar_try_wait(bars + 8 * i, i < slot ? phase : phase ^ 1u))
        if (globaltimer_ns() - t0 > kWaitLimitNs) break;
  }
  __device__ __forceinline__ void release() {
    __syncwarp();
    slot = slot + 1 == kSlots ? 0 : slot + 1;
    phase ^= slot == 0;
  }
};

// Launched as a programmatic dependent: waits for the kernel before it with griddepcontrol.wait.
template <typename... Args>
inline bool launch_dependent(void (*kernel)(Args...), int grid, int threads, size_t smem, cudaStream_t s,
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

}  // namespace
}  // namespace cmoe
