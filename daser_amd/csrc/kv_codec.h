// kv_codec.h -- element codecs of the re-rotation.
// Part of libdaser_kv.

#pragma once

#include "kv_common.h"

namespace {

// ---------------------------------------------------------------------------
// Element codecs for the rotation. Each 16-byte vector holds VE elements.

__device__ __forceinline__ float bf16_to_f32(uint32_t h) {
  return __uint_as_float(h << 16);
}
// Round-to-nearest-even fp32 -> bf16; NaN -> 0x7FC0 with its sign dropped.
__device__ __forceinline__ uint32_t f32_to_bf16(float f) {
  uint32_t u = __float_as_uint(f);
  if ((u & 0x7fffffffu) > 0x7f800000u) return 0x7fc0u;
  u += 0x7fffu + ((u >> 16) & 1u);
  return u >> 16;
}

__device__ __forceinline__ float fp16_to_f32(uint32_t h) {
  return (float)__builtin_bit_cast(_Float16, (uint16_t)h);
}
// fp32 -> fp16 by the hardware conversion (round-to-nearest-even) of the fp32
// value itself; NaN -> 0x7E00.
__device__ __forceinline__ uint32_t f32_to_fp16(float f) {
  if (__builtin_isnan(f)) return 0x7e00u;
  asm("" : "+v"(f));
  return (uint32_t)__builtin_bit_cast(uint16_t, (_Float16)f);
}
// a * b + t rounded once, to fp16: the vector kernels' fp16 sums. The compiler
// fuses the conversion in some kernels and not in others; by name, every kernel
// rounds alike, and once.
__device__ __forceinline__ uint32_t fma_fp16(float a, float b, float t) {
  _Float16 h;
  asm("v_fma_mixlo_f16 %0, %1, %2, %3" : "=v"(h) : "v"(a), "v"(b), "v"(t));
  return (uint32_t)__builtin_bit_cast(uint16_t, h);
}
// The two halves of w with NaN -> 0x7E00.
__device__ __forceinline__ uint32_t canonical_fp16(uint32_t w) {
  if ((w & 0x7fffu) > 0x7c00u) w = (w & 0xffff0000u) | 0x7e00u;
  if ((w & 0x7fff0000u) > 0x7c000000u) w = (w & 0xffffu) | 0x7e000000u;
  return w;
}

// OCP e4m3fn (bias 7, no infinities, S.1111.111 = NaN) through the gfx950
// conversion instructions, which use the OCP formats: v_cvt_pk_f32_fp8
// decodes two codes, v_cvt_pk_fp8_f32 encodes two floats with
// round-to-nearest-even (both checked exhaustively against the bit-level
// definition on MI355X: all 256 codes, 200k values incl. every midpoint).
// Encoding saturates by clamping to +-448 first (compare-select keeps NaN);
// the instruction turns NaN into 0xFF, which the clamp range never produces,
// so 0xFF bytes are rewritten to the canonical 0x7F.
typedef float f32x2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ float clamp448(float f) {
  f = f > 448.0f ? 448.0f : f;
  return f < -448.0f ? -448.0f : f;
}
// 0x80 in every byte of w that equals 0xFF.
__device__ __forceinline__ uint32_t ff_bytes(uint32_t w) {
  const uint32_t t = ~w;
  return ~(((t & 0x7f7f7f7fu) + 0x7f7f7f7fu) | t) & 0x80808080u;
}
__device__ __forceinline__ void e4m3x4_to_f32(uint32_t w, float* x) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
  x[0] = lo.x;
  x[1] = lo.y;
  x[2] = hi.x;
  x[3] = hi.y;
}
__device__ __forceinline__ uint32_t f32x4_to_e4m3(const float* y) {
  int e = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(y[0]), clamp448(y[1]), 0, false);
  e = __builtin_amdgcn_cvt_pk_fp8_f32(clamp448(y[2]), clamp448(y[3]), e, true);
  const uint32_t w = (uint32_t)e;
  return w ^ ff_bytes(w);
}

// OCP e5m2 (bias 15, infinities, S.11111.{01,10,11} = NaN) through the
// gfx950 bf8 conversions (v_cvt_pk_f32_bf8 / v_cvt_pk_bf8_f32, round to
// nearest even). Encoding saturates as for e4m3: finite values and
// infinities clamp to +-57344 (compare-select keeps NaN), so an encoded byte
// with an all-ones exponent is NaN, rewritten to torch's canonical 0x7F.
__device__ __forceinline__ float clamp57344(float f) {
  f = f > 57344.0f ? 57344.0f : f;
  return f < -57344.0f ? -57344.0f : f;
}
__device__ __forceinline__ void e5m2x4_to_f32(uint32_t w, float* x) {
  const f32x2 lo = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, false);
  const f32x2 hi = __builtin_amdgcn_cvt_pk_f32_bf8((int)w, true);
  x[0] = lo.x;
  x[1] = lo.y;
  x[2] = hi.x;
  x[3] = hi.y;
}
__device__ __forceinline__ uint32_t f32x4_to_e5m2(const float* y) {
  int e = __builtin_amdgcn_cvt_pk_bf8_f32(clamp57344(y[0]), clamp57344(y[1]), 0, false);
  e = __builtin_amdgcn_cvt_pk_bf8_f32(clamp57344(y[2]), clamp57344(y[3]), e, true);
  const uint32_t w = (uint32_t)e;
  // bytes whose exponent bits (0x7C) are all set: 0x80 in each such byte
  const uint32_t x = (w & 0x7c7c7c7cu) ^ 0x7c7c7c7cu;  // zero byte <=> exponent all ones
  const uint32_t nan = ~(((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x | 0x7f7f7f7fu);
  const uint32_t bytes = (nan >> 7) * 0xffu;
  return (w & ~bytes) | (0x7f7f7f7fu & bytes);
}

// The 8-bit formats: one byte per element, K scaled by the layer's k_scale.
template <int DT>
constexpr bool is_fp8() {
  return DT == DSR_DTYPE_FP8_E4M3 || DT == DSR_DTYPE_FP8_E5M2;
}

// The codecs' quick encoders round by the hardware's conversion alone, and say
// whether a result may need more (NaN, or a value outside the format): those
// vectors go through encode. A rotated page holds next to none of them.
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

template <int DT>
struct Codec;

template <>
struct Codec<DSR_DTYPE_BF16> {
  static constexpr int VE = 8;
  __device__ static void decode(u32x4 v, float* x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = bf16_to_f32(v[k] & 0xffffu);
      x[2 * k + 1] = bf16_to_f32(v[k] >> 16);
    }
  }
  __device__ static u32x4 encode(const float* y) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = f32_to_bf16(y[2 * k]) | (f32_to_bf16(y[2 * k + 1]) << 16);
    return v;
  }
  static constexpr uint32_t kSigns = 0x80008000u;
  __device__ static bool encode_quick(const float* y, u32x4* v) {
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x2 f = {y[2 * k], y[2 * k + 1]};
      const uint32_t w = __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
      odd |= (w & 0x7fff7fffu) + 0x007f007fu;  // past infinity: bit 15
      (*v)[k] = w;
    }
    return odd & kSigns;
  }
};

template <>
struct Codec<DSR_DTYPE_FP16> {
  static constexpr int VE = 8;
  __device__ static void decode(u32x4 v, float* x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = fp16_to_f32(v[k] & 0xffffu);
      x[2 * k + 1] = fp16_to_f32(v[k] >> 16);
    }
  }
  __device__ static u32x4 encode(const float* y) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k)
      v[k] = f32_to_fp16(y[2 * k]) | (f32_to_fp16(y[2 * k + 1]) << 16);
    return v;
  }
  static constexpr uint32_t kSigns = 0x80008000u;
  // the rotated sums x * c + t themselves; c: the cosine of element e is c[e / per].x
  template <int per>
  __device__ static u32x4 encode_sums(const float* x, const float2* c, const float* t) {
    u32x4 v;
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const int e = 2 * k;
      v[k] = fma_fp16(x[e], c[e / per].x, t[e]) |
             fma_fp16(x[e + 1], c[(e + 1) / per].x, t[e + 1]) << 16;
      odd |= (v[k] & 0x7fff7fffu) + 0x03ff03ffu;  // past infinity: bit 15
    }
    if (odd & kSigns)
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = canonical_fp16(v[k]);
    return v;
  }
};

template <>
struct Codec<DSR_DTYPE_FP8_E4M3> {
  static constexpr int VE = 16;
  __device__ static void decode(u32x4 v, float* x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) e4m3x4_to_f32(v[k], x + 4 * k);
  }
  __device__ static u32x4 encode(const float* y) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f32x4_to_e4m3(y + 4 * k);
    return v;
  }
  static constexpr uint32_t kSigns = 0x80808080u;
  // without the clamp, values past +-464 encode as NaN too
  __device__ static bool encode_quick(const float* y, u32x4* v) {
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int e = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k], y[4 * k + 1], 0, false);
      e = __builtin_amdgcn_cvt_pk_fp8_f32(y[4 * k + 2], y[4 * k + 3], e, true);
      odd |= ((uint32_t)e & 0x7f7f7f7fu) + 0x01010101u;  // 0x7F: bit 7
      (*v)[k] = (uint32_t)e;
    }
    return odd & kSigns;
  }
};

template <>
struct Codec<DSR_DTYPE_FP8_E5M2> {
  static constexpr int VE = 16;
  __device__ static void decode(u32x4 v, float* x) {
#pragma unroll
    for (int k = 0; k < 4; ++k) e5m2x4_to_f32(v[k], x + 4 * k);
  }
  __device__ static u32x4 encode(const float* y) {
    u32x4 v;
#pragma unroll
    for (int k = 0; k < 4; ++k) v[k] = f32x4_to_e5m2(y + 4 * k);
    return v;
  }
  static constexpr uint32_t kSigns = 0x80808080u;
  // without the clamp, values past the largest finite one encode as infinity
  __device__ static bool encode_quick(const float* y, u32x4* v) {
    uint32_t odd = 0;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      int e = __builtin_amdgcn_cvt_pk_bf8_f32(y[4 * k], y[4 * k + 1], 0, false);
      e = __builtin_amdgcn_cvt_pk_bf8_f32(y[4 * k + 2], y[4 * k + 3], e, true);
      odd |= ((uint32_t)e & 0x7c7c7c7cu) + 0x04040404u;  // exponent all ones: bit 7
      (*v)[k] = (uint32_t)e;
    }
    return odd & kSigns;
  }
};

}  // namespace
