// mc_paged.cuh -- what the paged serving operators share: activation types,
// the 4-bit page format and the host-side checks of their C entry points.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "mc_internal.cuh"
#include "modelc_cuda.h"

namespace mc {

mc_status set_error(mc_status st, const char* msg);  // mc_api.cu

// Checks, once a device, that it is an sm_100 device.
mc_status paged_check(int device);
int paged_sms(int device);  // its SM count (after paged_check)

// Makes a checked device current, and the caller's current again at the end of
// the scope; does nothing where they are the same.
class PagedDevice {
 public:
  explicit PagedDevice(int device);
  ~PagedDevice() {
    if (back_ >= 0) cudaSetDevice(back_);
  }
  PagedDevice(const PagedDevice&) = delete;
  PagedDevice& operator=(const PagedDevice&) = delete;
  mc_status status;

 private:
  int back_ = -1;
};

#define MC_PCK(call)                                                          \
  do {                                                                        \
    cudaError_t e_ = (call);                                                  \
    if (e_ != cudaSuccess)                                                    \
      return ::mc::set_error(e_ == cudaErrorMemoryAllocation ? MC_E_OOM : MC_E_CUDA, \
                             cudaGetErrorString(e_));                         \
  } while (0)
// For the rest of the function, or until it returns with the error.
#define MC_PAGED_DEVICE(device)         \
  ::mc::PagedDevice device_scope(device); \
  if (device_scope.status != MC_OK) return device_scope.status
#define MC_PCKS(expr)             \
  do {                            \
    mc_status s_ = (expr);        \
    if (s_ != MC_OK) return s_;   \
  } while (0)

inline bool aligned(const void* p, size_t n) { return ((uintptr_t)p % n) == 0; }

// ---------------------------------------------------------------------------
// The 4-bit page.  64 tokens of one key/value head in 72 D bytes (D = 64 or
// 128): K codes (64 rows of D/2 bytes), V codes, K scales, V scales (f16).
// Values follow the q4_0 rule of the weights: per 32 consecutive values
// d = (the value of largest size, first on ties) / -8, code = trunc(x/d + 8.5)
// in 0..15, value = (code - 8) f16(d).
//
// A row of D codes is W = D/8 words; value d sits in word d % W, nibble
// nib(d / W).  nib(2p) = p and nib(2p + 1) = p + 4, so that
// (word >> 8(p/2)) & (0x000f000f << 4(p%2)) has the codes of the values
// (2p W + w, (2p + 1) W + w), both in one block of 32, in its two halves, as
// the attention turns them into an f16 pair (an OR and one f16 operation).
// Tokens of D = 128 whose bit 1 is set hold the two 32-byte halves of a row
// swapped: the four rows a warp reads at once then lie in different banks.
// Scales are stored in the order in which the attention's lanes use them:
// [8 groups of 8 tokens][4 t][D/32 blocks][2 e], entry (t, b, e) for token
// kv4_token(2t + e) of the group.
// ---------------------------------------------------------------------------
constexpr int kKv4Page = 64;
__host__ __device__ constexpr int kv4_page_bytes(int D) { return 72 * D; }
// Tensor-core column n of a group of 8 tokens holds token kv4_token(n), its own inverse.
__host__ __device__ inline int kv4_token(int n) { return n < 4 ? n : n ^ 1; }
__host__ __device__ inline int kv4_nib(int i) { return (i >> 1) + 4 * (i & 1); }
// Index of block b of token s (0..63) in a page's K or V scales.
__host__ __device__ inline int kv4_scale_at(int s, int b, int NB) {
  const int n = kv4_token(s & 7);
  return (((s >> 3) * 4 + (n >> 1)) * NB + b) * 2 + (n & 1);
}
// Word index of logical word w in the row of token s.
template <int D>
__host__ __device__ inline int kv4_word_at(int s, int w) {
  return D == 128 ? w ^ ((s & 2) << 2) : w;
}

// ------------------------------------------------------------ type helpers
template <typename T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ float to_f<__half>(__half x) { return __half2float(x); }
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) { return __bfloat162float(x); }
template <typename T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) { return x; }
template <>
__device__ __forceinline__ __half from_f<__half>(float x) { return __float2half_rn(x); }
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// two f32 operations at once
__device__ __forceinline__ float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, c, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\tmov.b64 c, {%6, %7};\n\t"
      "fma.rn.f32x2 d, a, b, c;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
__device__ __forceinline__ float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 a, b, d;\n\t"
      "mov.b64 a, {%2, %3};\n\tmov.b64 b, {%4, %5};\n\t"
      "add.rn.f32x2 d, a, b;\n\tmov.b64 {%0, %1}, d;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// ------------------------------------------------- asynchronous copies
__device__ __forceinline__ uint32_t sm_ptr(const void* p) {
  return (uint32_t)__cvta_generic_to_shared(p);
}
__device__ __forceinline__ void bar_init(uint64_t* b, uint32_t n) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sm_ptr(b)), "r"(n) : "memory");
}
__device__ __forceinline__ void bar_expect(uint64_t* b, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(sm_ptr(b)), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ void bar_arrive(uint64_t* b) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sm_ptr(b)) : "memory");
}
__device__ __forceinline__ bool bar_try(uint64_t* b, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(sm_ptr(b)), "r"(parity)
      : "memory");
  return done != 0;
}
// Waits for the phase with this parity, two seconds at most: far above any
// copy's or product's time, so it runs out only when something else failed.
__device__ __forceinline__ bool bar_loop(uint32_t b, uint32_t parity) {
  unsigned long long t0 = 0, t1;
  for (int i = 0;; ++i) {
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(done)
        : "r"(b), "r"(parity)
        : "memory");
    if (done) return true;
    if (i % 64 == 63) {
      asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t1));
      if (!t0) t0 = t1;
      if (t1 - t0 > 2000000000ull) return false;
    }
  }
}
__device__ __forceinline__ bool bar_wait(uint64_t* b, uint32_t parity) { return bar_loop(sm_ptr(b), parity); }
// The same for a whole warp: true where no lane's wait ran out.
__device__ __forceinline__ bool warp_wait(uint64_t* b, uint32_t parity) {
  return __all_sync(~0u, bar_wait(b, parity));
}
// `bytes` (a multiple of 16) from global to shared memory, both 16-byte
// aligned, counted on an mbarrier of this block.
__device__ __forceinline__ void copy_bulk(void* dst, const void* src, uint32_t bytes, uint64_t* b) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          sm_ptr(dst)),
      "l"(src), "r"(bytes), "r"(sm_ptr(b))
      : "memory");
}

}  // namespace mc
