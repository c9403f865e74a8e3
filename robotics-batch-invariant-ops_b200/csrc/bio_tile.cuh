// Device and host helpers shared by the paged and the sliding-window
// attention: parked bounded waits, TMA boxes addressed in shared space, 2^x on
// the special-function unit, and tensor maps over 16-bit operands.
#pragma once

#include <type_traits>

#include "bio_common.cuh"

namespace bio {

// 2^x on the special-function unit (PTX ex2.approx: 2 ulp, 2^-inf = 0).
__device__ __forceinline__ float pow2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

__device__ __forceinline__ void expect_bytes(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0,
                                         int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(bar)
      : "memory");
}

// Bounded wait that polls without giving the warp up.
__device__ __forceinline__ bool spin_wait(uint32_t a, uint32_t parity, volatile int* abort_flag,
                                          int* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 0; i < kWaitMaxIters; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity)
        : "memory");
    if (done) return true;
    if ((i & 255u) != 255u) continue;
    if (t0 == 0) t0 = global_timer_ns();
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitTimeoutNs) break;
  }
  *abort_flag = 1;
  raise_status(status, BIO_DEV_TIMEOUT);
  return false;
}

// Bounded wait (the contract of mbar_wait) whose polls park the warp: polling
// warps take issue slots from the one or two that share their scheduler.
__device__ __forceinline__ bool parked_wait(uint32_t a, uint32_t parity,
                                            volatile int* abort_flag, int* status) {
  uint64_t t0 = 0;
  for (uint32_t i = 0; i < kWaitMaxIters; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(a), "r"(parity), "r"(100000u)
        : "memory");
    if (done) return true;
    if (i == 0) t0 = global_timer_ns();
    if (*abort_flag) return false;
    if (global_timer_ns() - t0 > kWaitTimeoutNs) break;
  }
  *abort_flag = 1;
  raise_status(status, BIO_DEV_TIMEOUT);
  return false;
}

// Division of 0 <= x < 2^31 by a fixed n >= 1: (mulhi(x, mul) + x) >> shift with
// 2^(shift-1) < n <= 2^shift and mul = floor(2^32 (2^shift - n) / n) + 1
// (Granlund and Montgomery, "Division by invariant integers using multiplication",
// 1994).
struct FixedDiv {
  unsigned mul, shift, n;
  __device__ __forceinline__ int quotient(int x) const {
    return static_cast<int>((__umulhi(static_cast<unsigned>(x), mul) + static_cast<unsigned>(x)) >>
                            shift);
  }
};

__host__ __device__ inline FixedDiv fixed_div(int64_t n) {
  FixedDiv d;
  d.n = static_cast<unsigned>(n);
  d.shift = 0;
  while ((1ull << d.shift) < static_cast<uint64_t>(n)) ++d.shift;
  d.mul = static_cast<unsigned>(((1ull << 32) * ((1ull << d.shift) - d.n)) / d.n + 1);
  return d;
}

}  // namespace bio

namespace bio_host {

// Tensor map {column, n1, n2, n3} of 16-bit elements with 128-byte swizzle and
// boxes of 64 x rows x rows2 x 1; element strides.  False for strides that no
// tensor map takes.
template <typename T>
inline bool map_of(CUtensorMap* map, const void* ptr, int64_t cols, int64_t n1, int64_t n2,
                   int64_t n3, int64_t s1, int64_t s2, int64_t s3, int rows, int rows2 = 1) {
  EncodeTiledFn enc = encode_tiled_fn();
  if (enc == nullptr) return false;
  const cuuint64_t dims[4] = {static_cast<cuuint64_t>(cols), static_cast<cuuint64_t>(n1),
                              static_cast<cuuint64_t>(n2), static_cast<cuuint64_t>(n3)};
  // the stride of a dimension of one element is never used, but has to be valid
  auto bytes = [](int64_t n, int64_t s) { return static_cast<cuuint64_t>(n > 1 ? 2 * s : 16); };
  const cuuint64_t strides[3] = {bytes(n1, s1), bytes(n2, s2), bytes(n3, s3)};
  const cuuint32_t box[4] = {64, static_cast<cuuint32_t>(rows),
                             static_cast<cuuint32_t>(rows2), 1},
                   ones[4] = {1, 1, 1, 1};
  return enc(map,
             std::is_same<T, __half>::value ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                            : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16,
             4, const_cast<void*>(ptr), dims, strides, box, ones, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace bio_host
