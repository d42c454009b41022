// 4-bit KV pools (FI_DTYPE_MXFP4): the format, its place in memory and its conversions.
//
// A head's row of D elements is D / 32 groups of 32 consecutive elements.  A group holds 32 e2m1
// codes (sign, two exponent bits, one mantissa bit: 0, 0.5, 1, 1.5, 2, 3, 4, 6) and one scale byte
// E: value = e2m1(code) * 2^(E - 127), 17 bytes for 32 elements.  Both factors are short, so every
// value is exact in bf16 and f32 and products with it need no rounding of the cache.
//
// The scale of a group with largest magnitude m is the smallest power of two s with m < 7 s: the
// top code 6 then takes (5 s, 7 s), half a step of its binade either side, so no value is off by
// more than half a step and none is cut off.  s lies in [2^-125, 2^125] (E in [2, 252]): below it
// values round to zero as below any smallest step, above it 6 s would pass f32's largest (a group
// with m >= 7 * 2^125 is cut off at 6 * 2^125).  Codes round to nearest, ties to the even code.
// A group with an infinity or a NaN has E = 255 and codes 0, and reads as NaN throughout.
#pragma once

#include <type_traits>

#include "fi_device.h"

namespace fi {

constexpr int kFp4Group = 32;  // elements that share a scale
constexpr uint32_t kFp4MaxScale = 252;  // the largest scale byte of values: 6 * 2^(E - 127) may be infinite above

// One pool array: codes [num_blocks][Hkv][block_size][D / 2] (element 2 i in the low half of byte
// i), then scales [num_blocks][Hkv][block_size][D / 32].  Codes and scales are apart so that a
// row's codes stay aligned to their size (16 bytes and up) for 16-byte loads.
__host__ __device__ inline size_t fp4_code_bytes(int64_t num_blocks, int hkv, int block_size, int d) {
  return static_cast<size_t>(num_blocks) * hkv * block_size * (d / 2);
}

__host__ __device__ inline size_t fp4_pool_bytes(int64_t num_blocks, int hkv, int block_size, int d) {
  return fp4_code_bytes(num_blocks, hkv, block_size, d) +
         static_cast<size_t>(num_blocks) * hkv * block_size * (d / kFp4Group);
}

#if defined(__HIPCC__)

// The largest magnitude of a group, as bits without the sign: integer order is the values' order,
// with infinities and NaN on top.
__device__ __forceinline__ uint32_t magnitude_bits(float x) { return __float_as_uint(x) & 0x7fffffffu; }

// The maximum over aligned groups of kLanes lanes (2, 4 or 8).
template <int kLanes>
__device__ __forceinline__ uint32_t group_max(uint32_t v) {
  static_assert(kLanes == 2 || kLanes == 4 || kLanes == 8, "group size");
  auto mov = [](uint32_t x, auto ctrl) {
    return static_cast<uint32_t>(
        __builtin_amdgcn_mov_dpp(static_cast<int>(x), decltype(ctrl)::value, 0xF, 0xF, false));
  };
  v = max(v, mov(v, std::integral_constant<int, 0xB1>{}));
  if constexpr (kLanes >= 4) v = max(v, mov(v, std::integral_constant<int, 0x4E>{}));
  if constexpr (kLanes >= 8) v = max(v, mov(v, std::integral_constant<int, 0x141>{}));
  return v;
}

// The scale byte of a group whose largest magnitude has bits `top`: exponent - 2, one more where
// the mantissa reaches 1.75 (m >= 7 * 2^(exponent - 2)).
__device__ __forceinline__ uint32_t fp4_scale(uint32_t top) {
  if (top >= 0x7f800000u) return 255u;
  const int e = static_cast<int>(top >> 23) - 2 + ((top & 0x7fffffu) >= 0x600000u ? 1 : 0);
  return static_cast<uint32_t>(min(max(e, 2), static_cast<int>(kFp4MaxScale)));
}

// A scale byte as the f32 whose exponent field it is (255: an infinity, which the conversions
// below turn into NaN for every code, zero among them).
__device__ __forceinline__ float fp4_scale_f32(uint32_t e) { return __uint_as_float(e << 23); }

// Codes of two values divided by the scale (nearest even, cut off at 6) into byte kByte of `old`.
// The instruction's results equal the format's rule for every scale byte from 2 to 252, ties, their
// neighbours, subnormals and values above 6 scales among them (tests/test_gpu_fp4_scales.py); non-finite
// groups do not come here.
template <int kByte>
__device__ __forceinline__ uint32_t fp4_pack2(uint32_t old, float a, float b, float scale) {
  return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(old, a, b, scale, kByte);
}

// The two values of byte kByte of `codes`, as packed bf16 (exact): element 2 i in the low half.
template <int kByte>
__device__ __forceinline__ uint32_t fp4_widen2(uint32_t codes, float scale) {
  return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(codes, scale, kByte));
}

// Eight values of one dword of codes as four packed bf16 pairs.
__device__ __forceinline__ uint4 fp4_widen8(uint32_t codes, float scale) {
  return make_uint4(fp4_widen2<0>(codes, scale), fp4_widen2<1>(codes, scale), fp4_widen2<2>(codes, scale),
                    fp4_widen2<3>(codes, scale));
}

__device__ __forceinline__ float4 bf16x4_to_f32(uint32_t lo, uint32_t hi) {
  return make_float4(bf16_bits_to_f32(lo & 0xffffu), bf16_bits_to_f32(lo >> 16), bf16_bits_to_f32(hi & 0xffffu),
                     bf16_bits_to_f32(hi >> 16));
}

// kBytes of codes from p, in one load (16, 8, 4, 2 or 1 bytes).
template <int kBytes>
struct Codes {
  uint32_t w[kBytes < 4 ? 1 : kBytes / 4];
  __device__ __forceinline__ void load(const uint8_t* p) {
    if constexpr (kBytes == 16) {
      const uint4 v = *reinterpret_cast<const uint4*>(p);
      w[0] = v.x;
      w[1] = v.y;
      w[2] = v.z;
      w[3] = v.w;
    } else if constexpr (kBytes == 8) {
      const uint2 v = *reinterpret_cast<const uint2*>(p);
      w[0] = v.x;
      w[1] = v.y;
    } else if constexpr (kBytes == 4) {
      w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (kBytes == 2) {
      w[0] = *reinterpret_cast<const uint16_t*>(p);
    } else {
      w[0] = *p;
    }
  }
};

// Eight consecutive elements of a group held by four neighbouring lanes: their codes, with the
// group's scale byte.
__device__ __forceinline__ uint32_t fp4_quantise8(const float4& lo, const float4& hi, uint32_t& scale_byte) {
  uint32_t top = max(max(max(magnitude_bits(lo.x), magnitude_bits(lo.y)), max(magnitude_bits(lo.z), magnitude_bits(lo.w))),
                     max(max(magnitude_bits(hi.x), magnitude_bits(hi.y)), max(magnitude_bits(hi.z), magnitude_bits(hi.w))));
  top = group_max<4>(top);
  scale_byte = fp4_scale(top);
  if (scale_byte == 255u) return 0u;
  const float s = fp4_scale_f32(scale_byte);
  uint32_t w = fp4_pack2<0>(0u, lo.x, lo.y, s);
  w = fp4_pack2<1>(w, lo.z, lo.w, s);
  w = fp4_pack2<2>(w, hi.x, hi.y, s);
  return fp4_pack2<3>(w, hi.z, hi.w, s);
}

#endif  // __HIPCC__

}  // namespace fi
