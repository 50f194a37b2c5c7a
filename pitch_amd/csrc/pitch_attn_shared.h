// What the attention translation units share: building blocks of the 16-bit matrix-core kernels (pitch_attn_codes.hip,
// pitch_paged_attn.hip), the kinds of caches and the launch interface of pitch_attn_codes.hip.
#pragma once

#include "pitch_device.h"

namespace pitch {

constexpr float kLn2 = 0x1.62e430p-1f;   // ln(2)

typedef float v4f __attribute__((ext_vector_type(4)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef uint32_t w4 __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) uint32_t lds_u32;
typedef uint32_t u32_any __attribute__((aligned(1)));

__device__ __forceinline__ v4f mfma_f16(w4 a, w4 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}
__device__ __forceinline__ v4f mfma_bf16(w4 a, w4 b, v4f c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
}

// Largest of a and b over the lane pair at distance 32 (16): of a in the lower lane of the pair, of b in the upper one.
__device__ __forceinline__ float max32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return fmax_hw(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
__device__ __forceinline__ float max16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return fmax_hw(__uint_as_float(r[0]), __uint_as_float(r[1]));
}
// Largest value over each row of 16 lanes, in all its lanes.
__device__ __forceinline__ float row_max(float x) {
  x = fmax_hw(x, xchg<1>(x));
  x = fmax_hw(x, xchg<2>(x));
  x = fmax_hw(x, xchg<4>(x));
  return fmax_hw(x, xchg<8>(x));
}
// A wave-uniform value, moved to a scalar register.
__device__ __forceinline__ float uniform(float x) {
  return __uint_as_float(__builtin_amdgcn_readfirstlane(__float_as_uint(x)));
}
__device__ __forceinline__ float lane_value(float x, int lane) {
  return __uint_as_float(__builtin_amdgcn_readlane(__float_as_uint(x), lane));
}
// Largest value over the wave (uniform).
__device__ __forceinline__ float wave_max(float x) { return lane_value(row_max(max16(max32(x, x), max32(x, x))), 0); }
// The same of four values: one reduction of a register whose rows hold the four.
__device__ __forceinline__ void wave_max4(const float (&x)[4], float (&m)[4]) {
  const float r = row_max(max16(max32(x[0], x[1]), max32(x[2], x[3])));
  m[0] = lane_value(r, 0);
  m[1] = lane_value(r, 32);
  m[2] = lane_value(r, 16);
  m[3] = lane_value(r, 48);
}
// The same of every head's value.
template <int NH>
__device__ __forceinline__ void wave_max_heads(const float (&x)[NH], float (&m)[NH]) {
#pragma unroll
  for (int h = 0; h < NH; h += 4) {
    const float x4[4] = {x[h], x[h + 1], x[h + 2], x[h + 3]};
    float m4[4];
    wave_max4(x4, m4);
#pragma unroll
    for (int k = 0; k < 4; ++k) m[h + k] = m4[k];
  }
}
__device__ __forceinline__ float wave_sum(float x) {
  x += xchg<1>(x);
  x += xchg<2>(x);
  x += xchg<4>(x);
  x += xchg<8>(x);
  {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  return x;
}
// (a, b) -> per lane, the sum of one operand over the lane pair at distance 32 (16): a for the lower lane of the
// pair, b for the upper one.
__device__ __forceinline__ float fold32(float a, float b) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
__device__ __forceinline__ float fold16(float a, float b) {
  const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
  return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}

// 2^e as a float32, -126 <= e <= 127.
__device__ __forceinline__ float pow2i(int e) { return __uint_as_float((uint32_t)(e + 127) << 23); }
// floor(log2 |x|) of a normal x (-127 for 0 and subnormals).
__device__ __forceinline__ int exponent_of(float x) { return (int)((__float_as_uint(x) >> 23) & 255u) - 127; }

__device__ __forceinline__ void wave_lds_fence() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The bits [pos, pos + width) of the lane's words w, moved to [at, at + width) of the result, with other bits around
// them (pos, width, at constants).
template <int NW>
__device__ __forceinline__ uint32_t bits_at(const uint32_t (&w)[NW], int pos, int width, int at) {
  const int wi = pos >> 5, q = pos & 31;
  if (q + width > 32) {
    const uint32_t next = w[wi + 1 < NW ? wi + 1 : wi];
    return q >= at ? __builtin_amdgcn_alignbit(next, w[wi], q - at) : (next << (at - q)) | (w[wi] >> (32 - (at - q)));
  }
  return q >= at ? w[wi] >> (q - at) : w[wi] << (at - q);
}

// b where the mask's bits are set, a elsewhere. (A choice between two elements of a private array by a lane's condition
// is compiled into an indexed load, which puts the array into scratch memory.)
__device__ __forceinline__ float pick(uint32_t mask, float a, float b) {
  return __uint_as_float((__float_as_uint(a) & ~mask) | (__float_as_uint(b) & mask));
}

// (x & mask) | rest in one instruction.
__device__ __forceinline__ uint32_t and_or(uint32_t x, uint32_t mask, uint32_t rest) {
  uint32_t r;
  asm("v_and_or_b32 %0, %1, %2, %3" : "=v"(r) : "v"(x), "s"(mask), "v"(rest));
  return r;
}

// Kinds of caches: key codec (with or without the key-bias term) and value codec.
#define kAttnKindTurbo 0      // TurboQuant keys and values
#define kAttnKindPolar 1      // PolarQuant keys and values
#define kAttnKindTurboBias 2  // the same with the key-bias term
#define kAttnKindPolarBias 3
#define kAttnKindChanTurbo 4  // per-channel keys, TurboQuant values
#define kAttnKindChanPolar 5  // per-channel keys, PolarQuant values
constexpr int kAttnKinds = 6;

#define PITCH_DECLARE_ATTN_CODES(K)                                                          \
  hipError_t launch_attn_codes_d64_k##K(const AttnArgs& a, uint32_t waves, hipStream_t s);   \
  hipError_t launch_attn_codes_d128_k##K(const AttnArgs& a, uint32_t waves, hipStream_t s);
PITCH_DECLARE_ATTN_CODES(0)
PITCH_DECLARE_ATTN_CODES(1)
PITCH_DECLARE_ATTN_CODES(2)
PITCH_DECLARE_ATTN_CODES(3)
PITCH_DECLARE_ATTN_CODES(4)
PITCH_DECLARE_ATTN_CODES(5)
#undef PITCH_DECLARE_ATTN_CODES

}  // namespace pitch
