// Device helpers shared by the bounded-cache attention kernels.
#pragma once

#include "fd_ptx.cuh"
#include "fd_stream.h"

namespace fd {

__device__ __forceinline__ StreamSeq sequence_of(const StreamParams& p, int b) {
  StreamSeq s;
  const int64_t cap = static_cast<int64_t>(p.max_blocks) << p.bs_log2;
  const int64_t n = load_index(p.sl, p.sl64, b * p.sls);
  s.n = static_cast<int>(min(max(n, int64_t(0)), cap));
  s.q0 = b;
  s.qlen = 1;
  if (p.qstart) {
    const int64_t a = load_index(p.qstart, p.qs64, b * p.qss);
    const int64_t z = load_index(p.qstart, p.qs64, (b + 1) * p.qss);
    const int64_t nt = p.num_tokens;
    const int64_t a1 = min(max(a, int64_t(0)), nt);
    s.q0 = static_cast<int>(a1);
    s.qlen = static_cast<int>(min(max(z, a1), nt) - a1);
  }
  return s;
}

// 8 elements of a strided row as one 16-byte value.
template <typename T>
__device__ __forceinline__ uint4 gather8(const T* src, int64_t stride) {
  __align__(16) T el[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) el[i] = src[i * stride];
  return *reinterpret_cast<const uint4*>(el);
}

// 16 bytes to shared memory (of which `bytes` are read, the rest is zero).
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, int bytes) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ void cp_async_commit() {
  asm volatile("cp.async.commit_group;" ::: "memory");
}
template <int N>
__device__ __forceinline__ void cp_async_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// Whether one of two packed 16-bit values is an infinity or NaN (all exponent
// bits set).
__device__ __forceinline__ bool nonfinite16(uint32_t w, uint32_t exp_mask) {
  return (w & exp_mask) == exp_mask || ((w >> 16) & exp_mask) == exp_mask;
}

}  // namespace fd
