// Device helpers of the block-scaled cache (e4m3 codes, scale 2^(e - 127)).
#pragma once

#include "common.cuh"
#include "sm100.cuh"

namespace mj {

__host__ __device__ __forceinline__ bool is_block_format(int kv_format) {
  return kv_format >= MJ_KV_FP8_B16 && kv_format <= MJ_KV_FP8_B128;
}
// log2 of the tokens of a block
__host__ __device__ __forceinline__ int block_log2(int kv_format) { return kv_format - MJ_KV_FP8_B16 + 4; }

// e as a reader takes it
__device__ __forceinline__ int block_e(unsigned char b) {
  return min(max((int)b, MJ_BLOCK_E_MIN), MJ_BLOCK_E_MAX);
}
__device__ __forceinline__ float block_scale(unsigned char b) { return __uint_as_float((uint32_t)block_e(b) << 23); }

// 8 elements to a 16-byte aligned address
__device__ __forceinline__ void store8(float* p, const float* v) {
  reinterpret_cast<float4*>(p)[0] = make_float4(v[0], v[1], v[2], v[3]);
  reinterpret_cast<float4*>(p)[1] = make_float4(v[4], v[5], v[6], v[7]);
}
__device__ __forceinline__ void store8(__nv_bfloat16* p, const float* v) {
  uint4 raw;
  __nv_bfloat162* e = reinterpret_cast<__nv_bfloat162*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
__device__ __forceinline__ void store8(__half* p, const float* v) {
  uint4 raw;
  __half2* e = reinterpret_cast<__half2*>(&raw);
#pragma unroll
  for (int i = 0; i < 4; ++i) e[i] = __floats2half2_rn(v[2 * i], v[2 * i + 1]);
  *reinterpret_cast<uint4*>(p) = raw;
}
// 32 bytes at a 32-byte aligned address
__device__ __forceinline__ void store32(void* p, uint4 a, uint4 b) {
  asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(a.x), "r"(a.y), "r"(a.z), "r"(a.w), "r"(b.x),
               "r"(b.y), "r"(b.z), "r"(b.w)
               : "memory");
}

// 8 elements of a row as they are in memory
template <typename T>
struct Raw8 {
  uint4 v[sizeof(T) / 2];
  __device__ __forceinline__ void load(const T* p, bool vec) {
    if (vec) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) / 2; ++i) v[i] = reinterpret_cast<const uint4*>(p)[i];
    } else {
      T* e = reinterpret_cast<T*>(v);
#pragma unroll
      for (int i = 0; i < 8; ++i) e[i] = p[i];
    }
  }
  __device__ __forceinline__ void get(float* x) const {
    const T* e = reinterpret_cast<const T*>(v);
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = (float)e[i];
  }
};
// 0x80 in every byte of w that is a NaN code (0x7F or 0xFF)
__device__ __forceinline__ uint32_t nan_codes(uint32_t w) { return ((w & 0x7F7F7F7Fu) + 0x01010101u) & 0x80808080u; }
// 16 codes with NaN made zero; true if one was
__device__ __forceinline__ bool drop_nan_codes(uint4& c) {
  const uint32_t x = nan_codes(c.x), y = nan_codes(c.y), z = nan_codes(c.z), w = nan_codes(c.w);
  if (!(x | y | z | w)) return false;
  c.x &= ~((x >> 7) * 0xFFu);
  c.y &= ~((y >> 7) * 0xFFu);
  c.z &= ~((z >> 7) * 0xFFu);
  c.w &= ~((w >> 7) * 0xFFu);
  return true;
}

// 8 values times f -> e4m3 codes: nearest even, saturating, NaN stays NaN
__device__ __forceinline__ uint2 quantize8(const float* v, float f) {
  uint16_t c[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 x = sm100::fmul2(make_float2(v[2 * i], v[2 * i + 1]), make_float2(f, f));
    c[i] = sm100::f2_to_e4m3x2(x.x, x.y);
  }
  return make_uint2(c[0] | ((uint32_t)c[1] << 16), c[2] | ((uint32_t)c[3] << 16));
}
__device__ __forceinline__ void dequantize8(uint2 codes, float f, float* v) {
  const uint16_t c[4] = {(uint16_t)codes.x, (uint16_t)(codes.x >> 16), (uint16_t)codes.y, (uint16_t)(codes.y >> 16)};
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const float2 p = sm100::e4m3x2_to_f2(c[i]);
    v[2 * i] = p.x * f, v[2 * i + 1] = p.y * f;
  }
}
// 4 codes times f, as codes
__device__ __forceinline__ uint32_t scale4(uint32_t codes, float f) {
  const float2 a = sm100::e4m3x2_to_f2((uint16_t)codes), b = sm100::e4m3x2_to_f2((uint16_t)(codes >> 16));
  return sm100::f2_to_e4m3x2(a.x * f, a.y * f) | ((uint32_t)sm100::f2_to_e4m3x2(b.x * f, b.y * f) << 16);
}

}  // namespace mj
