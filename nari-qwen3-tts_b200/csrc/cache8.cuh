// The 8-bit paged KV cache: its layout, its codes and their conversions.
//
// One layer is `cache` [pages, 2, P, Hkv, D] of one-byte codes (kind 0 = K,
// 1 = V), with one fp32 scale for every block of 16 tokens of a page, kind
// and KV head in `scales` [pages, 2, P / 16, Hkv]; an element stands for
// code * scale.  Codes are two's-complement int8 in [-127, 127] or e4m3.
// A block is what one TMA box of the attention kernels brings, so a tile of
// 16 tokens has one scale for K and one for V.
//
// The attention kernels multiply codes, exactly converted to 16-bit floats
// (both kinds of code fit fp16 and bf16 without rounding), and apply the
// scales to the fp32 scores and probabilities: no key or value is rounded
// again on its way to the tensor cores.
#pragma once

#include <cuda_fp8.h>
#include <cudaTypedefs.h>

#include <mutex>

#include "common.cuh"
#include "fp8.cuh"

namespace nqt {
namespace c8 {

constexpr int kBlock = 16;  // tokens that share a scale

template <bool E4M3>
__host__ __device__ constexpr float top_code() {
  return E4M3 ? 448.f : 127.f;
}

inline bool valid_code(int code) { return code == NQT_I8 || code == NQT_E4M3; }

// ---- codes -> numbers --------------------------------------------------------------
// Two int8 codes in bytes SEL_LO and SEL_HI of `biased` (= the four codes with their sign bits flipped) as
// f16x2: a byte u behind 0x64 is the f16 number 1024 + u, so subtracting 1152 leaves u - 128, exactly.
template <int SEL>
__device__ __forceinline__ uint32_t i8_pair_to_f16x2(uint32_t biased) {
  const uint32_t raw = __byte_perm(biased, 0x64646464u, SEL);
  const uint32_t off = 0x64806480u;  // 1152, 1152
  __half2 r = __hsub2(*reinterpret_cast<const __half2*>(&raw), *reinterpret_cast<const __half2*>(&off));
  return *reinterpret_cast<uint32_t*>(&r);
}

__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint16_t v) {
  uint32_t r;
  asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
  return r;
}

// Four codes of a word -> two f16x2: (bytes 0, 1) and (bytes 2, 3).
template <bool E4M3>
__device__ __forceinline__ void codes_to_f16_rows(uint32_t w, uint32_t& lo, uint32_t& hi) {
  if (E4M3) {
    lo = e4m3x2_to_f16x2(static_cast<uint16_t>(w));
    hi = e4m3x2_to_f16x2(static_cast<uint16_t>(w >> 16));
  } else {
    const uint32_t b = w ^ 0x80808080u;
    lo = i8_pair_to_f16x2<0x4140>(b);
    hi = i8_pair_to_f16x2<0x4342>(b);
  }
}

// Four codes of a word -> two f16x2: (bytes 0, 2) and (bytes 1, 3).
template <bool E4M3>
__device__ __forceinline__ void codes_to_f16_cols(uint32_t w, uint32_t& even, uint32_t& odd) {
  if (E4M3) {
    const uint32_t s = __byte_perm(w, 0u, 0x3120);
    even = e4m3x2_to_f16x2(static_cast<uint16_t>(s));
    odd = e4m3x2_to_f16x2(static_cast<uint16_t>(s >> 16));
  } else {
    const uint32_t b = w ^ 0x80808080u;
    even = i8_pair_to_f16x2<0x4240>(b);
    odd = i8_pair_to_f16x2<0x4341>(b);
  }
}

// Byte `i` of `w` as a number.
template <bool E4M3>
__device__ __forceinline__ float code_to_f32(uint32_t w, int i) {
  const uint32_t byte = (w >> (8 * i)) & 0xffu;
  if (E4M3) {
    const __half_raw h = __nv_cvt_fp8_to_halfraw(static_cast<__nv_fp8_storage_t>(byte), __NV_E4M3);
    return __half2float(__half(h));
  }
  return static_cast<float>(static_cast<int8_t>(byte));
}

// ---- numbers -> codes --------------------------------------------------------------
// Nearest code (ties to even) of x, saturating; NaN becomes code 0 as int8 and the NaN code as e4m3.
template <bool E4M3>
__device__ __forceinline__ uint32_t f32_to_code(float x) {
  if (E4M3) return static_cast<uint32_t>(__nv_cvt_float_to_fp8(x, __NV_SATFINITE, __NV_E4M3));
  if (x != x) return 0u;
  return static_cast<uint32_t>(__float2int_rn(fminf(fmaxf(x, -127.f), 127.f))) & 0xffu;
}

// Two codes, the first in the low byte.
template <bool E4M3>
__device__ __forceinline__ uint16_t codes_of_pair(float a, float b) {
  if (E4M3) return __nv_cvt_float2_to_fp8x2(make_float2(a, b), __NV_SATFINITE, __NV_E4M3);
  return static_cast<uint16_t>(f32_to_code<false>(a) | (f32_to_code<false>(b) << 8));
}

// ---- host --------------------------------------------------------------------------
inline PFN_cuTensorMapEncodeTiled_v12000 get_encode() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Shape checks that every entry point over an 8-bit layer shares.
inline int check_layer(const void* cache, const float* scales, int total_pages, int page_size, int hkv, int head_dim,
                       int code) {
  if (!cache || !scales || total_pages < 1 || hkv < 1) return NQT_ERR_ARG;
  if (!valid_code(code)) return NQT_ERR_UNSUPPORTED;
  if (head_dim != 64 && head_dim != 128) return NQT_ERR_UNSUPPORTED;
  if (page_size < kBlock || page_size % kBlock || page_size > 256 || hkv > 256) return NQT_ERR_UNSUPPORTED;
  if ((reinterpret_cast<uintptr_t>(cache) & 15) || (reinterpret_cast<uintptr_t>(scales) & 3)) return NQT_ERR_ARG;
  if (static_cast<int64_t>(total_pages) * 2 >= (int64_t(1) << 31)) return NQT_ERR_UNSUPPORTED;
  return NQT_OK;
}

}  // namespace c8
}  // namespace nqt
