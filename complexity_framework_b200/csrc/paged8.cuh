// Device helpers shared by the 8-bit paged KV cache kernels.
#pragma once
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include <atomic>

#include "common.cuh"
#include "paged8.h"

namespace cfb {

template <typename T>
struct P8Io;
template <>
struct P8Io<__nv_bfloat16> {
  static constexpr bool kBf16 = true;
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ __nv_bfloat16 cast(float a) { return __float2bfloat16(a); }
};
template <>
struct P8Io<__half> {
  static constexpr bool kBf16 = false;
  static __device__ __forceinline__ float2 unpack(uint32_t u) {
    return __half22float2(*reinterpret_cast<__half2*>(&u));
  }
  static __device__ __forceinline__ uint32_t pack(float a, float b) {
    __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  static __device__ __forceinline__ __half cast(float a) { return __float2half(a); }
};

template <int FMT>
__device__ __forceinline__ constexpr float p8_levels() {
  return FMT == kP8Int8 ? 127.f : 448.f;
}

// Four codes (one word) as two f16x2: (byte 0, byte 1) and (byte 2, byte 3).  Exact:
// an e4m3 number is an f16 number; an int8 code with its sign bit flipped is the low
// byte of the f16 number 1024 + 128 + code.
template <int FMT>
__device__ __forceinline__ void p8_to_half(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if constexpr (FMT == kP8Int8) {
    w ^= 0x80808080u;
    const __half2 bias = __half2half2(__ushort_as_half(0x6480));  // 1152
    uint32_t a = __byte_perm(w, 0x64646464u, 0x4140);
    uint32_t b = __byte_perm(w, 0x64646464u, 0x4342);
    __half2 x = __hsub2(*reinterpret_cast<__half2*>(&a), bias);
    __half2 y = __hsub2(*reinterpret_cast<__half2*>(&b), bias);
    lo = *reinterpret_cast<uint32_t*>(&x);
    hi = *reinterpret_cast<uint32_t*>(&y);
  } else {
    asm("{\n .reg .b16 l, h;\n mov.b32 {l, h}, %2;\n cvt.rn.f16x2.e4m3x2 %0, l;\n"
        " cvt.rn.f16x2.e4m3x2 %1, h;\n}"
        : "=r"(lo), "=r"(hi)
        : "r"(w));
  }
}

template <int FMT>
__device__ __forceinline__ void p8_to_float(uint32_t w, float* f) {
  uint32_t lo, hi;
  p8_to_half<FMT>(w, lo, hi);
  const float2 a = __half22float2(*reinterpret_cast<__half2*>(&lo));
  const float2 b = __half22float2(*reinterpret_cast<__half2*>(&hi));
  f[0] = a.x;
  f[1] = a.y;
  f[2] = b.x;
  f[3] = b.y;
}

// Four scaled values, finite and |f| <= levels up to rounding, to codes: to nearest, ties to
// even.  int8 rounds in the adder: f + 1.5 * 2^23 has the integer in its low byte: no
// conversion, and byte permutations gather the codes.
template <int FMT>
__device__ __forceinline__ uint32_t p8_from_float(const float* f) {
  if constexpr (FMT == kP8Int8) {
    constexpr float kRound = 12582912.f;
    const float2 ab = add2(make_float2(f[0], f[1]), make_float2(kRound, kRound));
    const float2 cd = add2(make_float2(f[2], f[3]), make_float2(kRound, kRound));
    return __byte_perm(
        __byte_perm(__float_as_uint(ab.x), __float_as_uint(ab.y), 0x0040),
        __byte_perm(__float_as_uint(cd.x), __float_as_uint(cd.y), 0x0040), 0x5410);
  } else {
    const uint32_t lo = __nv_cvt_float2_to_fp8x2(make_float2(f[0], f[1]), __NV_SATFINITE,
                                                 __NV_E4M3);
    const uint32_t hi = __nv_cvt_float2_to_fp8x2(make_float2(f[2], f[3]), __NV_SATFINITE,
                                                 __NV_E4M3);
    return lo | (hi << 16);
  }
}

// Kernels of these operators are launched with programmatic stream serialisation: their
// launch overlaps the end of the kernel before, whose results they may read after the wait.
__device__ __forceinline__ void p8_grid_wait() {
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
}

template <typename... KArgs, typename... Args>
int p8_launch(void (*kern)(KArgs...), dim3 grid, int threads, int smem, cudaStream_t stream,
              Args... args) {
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  cfg.stream = stream;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  return static_cast<int>(cudaLaunchKernelEx(&cfg, kern, static_cast<KArgs>(args)...));
}

// Opts a kernel in to its shared memory, once for each device.
template <auto Kern>
int p8_opt_in(int smem) {
  static std::atomic<uint64_t> done{0};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return static_cast<int>(e);
  const uint64_t bit = 1ull << (dev & 63);
  if (dev < 64 && (done.load(std::memory_order_relaxed) & bit)) return 0;
  e = cudaFuncSetAttribute(Kern, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) return static_cast<int>(e);
  if (dev < 64) done.fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

// A page id read from a table; one outside the pool is reported and read as page 0.
__device__ __forceinline__ int64_t p8_checked(int p, int64_t num_pages, int* err, int site) {
  if (static_cast<uint32_t>(p) >= static_cast<uint64_t>(num_pages)) {
    report_error(err, kErrBounds, site);
    return 0;
  }
  return p;
}
__device__ __forceinline__ int64_t p8_page(const int32_t* row, int i, int64_t num_pages, int* err,
                                           int site) {
  return p8_checked(__ldg(row + i), num_pages, err, site);
}

// Cached length of a sequence, held to what its page-table row can describe.
__device__ __forceinline__ int p8_len(const int32_t* kv_lens, int seq, int max_pages, int* err,
                                      int site) {
  const int n = __ldg(kv_lens + seq);
  if (n < 0 || n > max_pages * kP8Page) {
    report_error(err, kErrBounds, site);
    return n < 0 ? 0 : max_pages * kP8Page;
  }
  return n;
}

}  // namespace cfb
