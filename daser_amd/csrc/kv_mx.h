// kv_mx.h -- quantised records (OCP microscaling formats): the elements' codecs and the
// kernels that write records from the paged caches and read them back, by page and by
// token.
// Part of libdaser_kv.
//
// A block of 32 elements of one (token, head) row is held as q_i 2^(s - 127). With a =
// max |x_i|, s is the smallest code with a <= T 2^(s - 127), T the format's largest
// value and half its last step (127.5 / 64, 7): a clipped element is then off by no more
// than a rounded one may be. On N(0, 1) blocks e2m1 is off by 0.1118 sigma (rms) that
// way, by 0.1149 under the rule floor(log2 a) and 0.1154 where nothing may clip.
// Scaling by powers of two is exact, so there is one rounding, to the nearest code.
//
// Records hold a page head by head ([H][block_size][D]), whatever the cache's order: a
// head's tokens lie in one run, which attention over records reads whole.

#pragma once

#include "kv_codec.h"
#include "kv_flat.h"

namespace {

inline int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }

// Section bytes of one half; false for geometries that the format does not take.
inline bool mx_sections(int format, int block, int heads, int dim, int64_t* codes, int64_t* scales) {
  if (block <= 0 || heads <= 0 || dim <= 0 || dim % 32) return false;
  const __int128 elems = (__int128)block * heads * dim;
  if (elems * 2 > 0x7fffffffLL) return false;  // one buffer descriptor per cache page
  *codes = pad16((int64_t)elems / (format == DSR_MX_FP4 ? 2 : 1));
  *scales = pad16((int64_t)elems / 32);
  return true;
}

struct MxArgs {
  const uint64_t* layer_base;
  int64_t kv_stride, page_stride, num_blocks;
  uint8_t* staging;
  int64_t staging_bytes, layer_bytes, need;  // need: bytes of a layer in use
  int64_t page_bytes;                        // of a cache page
  int32_t layer0, first;  // table layers first ... are moved, record layers layer0 + l
  int32_t vecs;           // 16-byte vectors (8 elements) of a page
  int32_t codes, scales;  // section bytes of one half
  int32_t heads, block;
  int32_t block_shift;    // log2 of block, or -1
  FastDiv row_vecs, by_block, by_heads;  // vectors per row; block; heads
};

// Between a wave's writes to its part of the LDS and other lanes' reads, and before it is
// written again. The hardware keeps a wave's LDS operations in order; this is for the compiler.
__device__ __forceinline__ void wave_lds() {
  __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
  __builtin_amdgcn_wave_barrier();
  __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
}

// The rotation of a load's K.
struct MxRope {
  const float2* cos_sin;
  const int32_t* rope_idx;  // null: nothing is rotated
  const int32_t* layer_group;
  int32_t n_tables, n_groups;
  int32_t rot_vecs, half_vecs;  // rotated vectors of a row; neox: to the partner
};

template <int FMT>
__device__ __forceinline__ constexpr int mx_code_bytes() {  // of 8 elements
  return FMT == DSR_MX_FP4 ? 4 : 8;
}

// E8M0 code of a block whose largest magnitude has these fp32 bits.
template <int FMT>
__device__ __forceinline__ uint32_t mx_scale_code(uint32_t bits) {
  // bits + add carries into the exponent where the significand is past T's
  constexpr uint32_t add = FMT == DSR_MX_FP4 ? 0x1fffffu : 0x00ffffu;
  constexpr int sub = FMT == DSR_MX_FP4 ? 2 : 0;
  const int s = (int)((bits + add) >> 23) - sub;
  return bits >= 0x7f800000u ? 255u : (uint32_t)(s < 0 ? 0 : s);
}

// 2^(s - 127) for s < 255.
__device__ __forceinline__ float mx_scale(uint32_t s) {
  return __uint_as_float(s ? s << 23 : 0x00400000u);
}

typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

// fp32 bits of the largest magnitude of the 4 lanes' 8 elements each (one block);
// 0x7F800000 and up: one of them is not finite.
template <int DT>
__device__ __forceinline__ uint32_t mx_block_max(u32x4 v) {
  u16x2 m = __builtin_bit_cast(u16x2, v[0] & 0x7fff7fffu);
#pragma unroll
  for (int k = 1; k < 4; ++k)
    m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, v[k] & 0x7fff7fffu));
  uint32_t a = m.x > m.y ? m.x : m.y;
  const uint32_t b = (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0xb1, 0xf, 0xf, true);
  a = a > b ? a : b;
  const uint32_t c = (uint32_t)__builtin_amdgcn_mov_dpp((int)a, 0x4e, 0xf, 0xf, true);
  a = a > c ? a : c;
  if (DT == DSR_DTYPE_BF16) return a << 16;
  return a >= 0x7c00u ? 0x7f800000u : __float_as_uint(fp16_to_f32(a));
}

// 8 elements of a cache vector as codes under scale code s.
template <int FMT, int DT>
__device__ __forceinline__ uint2 mx_encode(u32x4 v, uint32_t s) {
  uint2 o{0u, 0u};
  if (FMT == DSR_MX_FP4) {
    const float scale = mx_scale(s);
// (the pair in a variable of its own: a bit cast of a vector's element takes the first)
#define DSR_FP4(K)                                                                             \
  {                                                                                            \
    const uint32_t w = v[K];                                                                   \
    if (DT == DSR_DTYPE_BF16)                                                                  \
      o.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(o.x, __builtin_bit_cast(bf16x2, w), scale, \
                                                      K);                                      \
    else                                                                                       \
      o.x = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(o.x, __builtin_bit_cast(f16x2, w), scale, K); \
  }
    DSR_FP4(0)
    DSR_FP4(1)
    DSR_FP4(2)
    DSR_FP4(3)
#undef DSR_FP4
  } else {
    float x[8];
    Codec<DT>::decode(v, x);
    uint32_t b[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      float y = __builtin_ldexpf(x[e], 133 - (int)s);
      y = __builtin_fminf(__builtin_fmaxf(y, -127.0f), 127.0f);
      b[e] = __float_as_uint(y + 12582912.0f);  // 1.5 * 2^23: the low byte is rne(y)
    }
    const uint32_t l = __builtin_amdgcn_perm(b[1], b[0], 0x0c0c0400u);
    const uint32_t h = __builtin_amdgcn_perm(b[3], b[2], 0x04000c0cu);
    o.x = l | h;
    o.y = __builtin_amdgcn_perm(b[5], b[4], 0x0c0c0400u) |
          __builtin_amdgcn_perm(b[7], b[6], 0x04000c0cu);
  }
  if (s == 255u) o = uint2{0u, 0u};
  return o;
}

// Bytes 2 h and 2 h + 1 of w, as int8, times p. A byte u = q + 128 behind 0x64 is the fp16
// number 1,024 + u, and a fused step takes fp16 in: q p = (1,024 + u) p - 1,152 p, exact. One
// permutation and two steps for two elements; a conversion for each was one more.
__device__ __forceinline__ f32x2 int8_pair(uint32_t w, int h, float p, float bias) {
  const uint32_t v = __builtin_amdgcn_perm(0x64646464u, w ^ 0x80808080u,
                                           h ? 0x04030402u : 0x04010400u);
  const f16x2 f = __builtin_bit_cast(f16x2, v);
  return {__builtin_fmaf((float)f.x, p, bias), __builtin_fmaf((float)f.y, p, bias)};
}

// Values of 8 codes under scale code s, NaN under 255.
template <int FMT>
__device__ __forceinline__ void mx_decode(uint2 c, uint32_t s, float* x) {
  if (FMT == DSR_MX_FP4) {
    const float scale = mx_scale(s);
    f32x2 f[4];
    f[0] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, scale, 0);
    f[1] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, scale, 1);
    f[2] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, scale, 2);
    f[3] = __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(c.x, scale, 3);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      x[2 * k] = f[k].x;
      x[2 * k + 1] = f[k].y;
    }
  } else {
    const float p = __builtin_ldexpf(1.0f, (int)s - 133), bias = -1152.0f * p;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x2 f = int8_pair(k < 2 ? c.x : c.y, k & 1, p, bias);
      x[2 * k] = f.x;
      x[2 * k + 1] = f.y;
    }
  }
  if (__builtin_expect(s >= 250u, 0)) {  // 1,152 p is past fp32, and 255 is NaN
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      if (FMT == DSR_MX_INT8)
        x[e] = __builtin_ldexpf((float)(int8_t)((e < 4 ? c.x : c.y) >> (8 * (e & 3))), (int)s - 133);
      if (s == 255u) x[e] = __uint_as_float(0x7fc00000u);
    }
  }
}

// Scale codes above it may read as more than the type holds, and 255 as NaN.
template <int FMT, int DT>
__device__ __forceinline__ constexpr uint32_t top_scale() {
  return DT == DSR_DTYPE_BF16 ? (FMT == DSR_MX_FP4 ? 252u : 249u)
                              : (FMT == DSR_MX_FP4 ? 140u : 141u);
}

// Two floats as the type, round to nearest even.
template <int DT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
  const f32x2 f = {x, y};
  if constexpr (DT == DSR_DTYPE_BF16)
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, bf16x2));
  else
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f, f16x2));
}

// 8 codes under scale code s as 8 values of the type; above top_scale()
// dequantise_any(). e2m1 has an instruction for it.
template <int FMT, int DT>
__device__ __forceinline__ u32x4 dequantise(const uint32_t* w, uint32_t s) {
  u32x4 o;
  if constexpr (FMT == DSR_MX_FP4) {
    const float scale = mx_scale(s);
#define DSR_DQ(K)                                                                            \
  if constexpr (DT == DSR_DTYPE_BF16)                                                        \
    o[K] = __builtin_bit_cast(uint32_t,                                                      \
                              __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w[0], scale, K));    \
  else                                                                                       \
    o[K] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(w[0], scale, K));
    DSR_DQ(0)
    DSR_DQ(1)
    DSR_DQ(2)
    DSR_DQ(3)
#undef DSR_DQ
  } else {
    const float p = __builtin_ldexpf(1.0f, (int)s - 133), bias = -1152.0f * p;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const f32x2 x = int8_pair(w[k >> 1], k & 1, p, bias);
      o[k] = pack2<DT>(x.x, x.y);
    }
  }
  return o;
}

// The same for any scale code: saturated; NaN under 255.
template <int FMT, int DT>
__device__ __forceinline__ u32x4 dequantise_any(const uint32_t* w, uint32_t s) {
  float x[8];
  mx_decode<FMT>(uint2{w[0], FMT == DSR_MX_FP4 ? 0u : w[1]}, s, x);
  constexpr uint32_t top = DT == DSR_DTYPE_BF16 ? 0x7f7f7f7fu : 0x7bff7bffu;
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    const uint32_t p = pack2<DT>(x[2 * k], x[2 * k + 1]), mag = p & 0x7fff7fffu;
    const u16x2 m = __builtin_elementwise_min(__builtin_bit_cast(u16x2, mag),
                                              __builtin_bit_cast(u16x2, top));
    v[k] = s == 255u ? (DT == DSR_DTYPE_BF16 ? 0x7fc07fc0u : 0x7e007e00u)
                     : (p & 0x80008000u) | __builtin_bit_cast(uint32_t, m);
  }
  return v;
}

// 8 floats as a cache vector; odd: they may be NaN or past the type's largest, where the
// vector is made with care (saturated, NaN canonical).
template <int DT>
__device__ __forceinline__ u32x4 mx_store_vec(float* y, bool odd) {
  u32x4 v;
#pragma unroll
  for (int k = 0; k < 4; ++k) v[k] = pack2<DT>(y[2 * k], y[2 * k + 1]);
  if (__builtin_expect(odd, 0)) {
    const float top = DT == DSR_DTYPE_BF16 ? __uint_as_float(0x7f7f0000u) : 65504.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      y[e] = y[e] > top ? top : y[e];
      y[e] = y[e] < -top ? -top : y[e];
    }
    v = Codec<DT>::encode(y);
  }
  return v;
}

// One half (K or V) of a record's layer.
struct MxHalf {
  const uint8_t* codes;
  const uint8_t* scales;
};
__device__ __forceinline__ MxHalf mx_half(const MxArgs& a, const uint8_t* rec, int half) {
  return {rec + (int64_t)half * a.codes, rec + 2 * (int64_t)a.codes + (int64_t)half * a.scales};
}

template <int FMT>
__device__ __forceinline__ uint2 mx_load_codes(const MxHalf& h, int vec) {
  if (FMT == DSR_MX_FP4)
    return uint2{__builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(h.codes) + vec), 0u};
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  const u32x2 w = __builtin_nontemporal_load(reinterpret_cast<const u32x2*>(h.codes) + vec);
  return uint2{w[0], w[1]};
}

// One vector (8 elements) of a record as loaded; K of a moved page: its neox partner's too.
struct MxVec {
  uint2 own, other;
  uint32_t s, s_other;
};
template <int FMT>
__device__ __forceinline__ MxVec mx_load_vec(const MxHalf& half, int rv, int partner) {
  MxVec v;
  v.own = mx_load_codes<FMT>(half, rv);
  v.s = half.scales[rv >> 2];
  if (partner >= 0) {
    v.other = mx_load_codes<FMT>(half, partner);
    v.s_other = half.scales[partner >> 2];
  }
  return v;
}
// As a cache vector, not rotated.
template <int FMT, int DT>
__device__ __forceinline__ u32x4 mx_plain_vec(const MxVec& v) {
  const uint32_t w[2] = {v.own.x, v.own.y};
  u32x4 o = dequantise<FMT, DT>(w, v.s);
  if (__builtin_expect(v.s > top_scale<FMT, DT>(), 0)) o = dequantise_any<FMT, DT>(w, v.s);
  return o;
}
// Rotated: c is the vector's column in its row, t its pairs' (cos, sin) two by two (neox 4,
// gptj 2 of them). The sines' products are rounded and the sums fused, as everywhere.
template <int FMT, int DT, int STYLE>
__device__ __forceinline__ u32x4 mx_turned_vec(const MxVec& v, int c, const MxRope& r,
                                               const f32x4* t) {
  float x[8];
  mx_decode<FMT>(v.own, v.s, x);
  bool odd = v.s >= top_scale<FMT, DT>();  // sums reach 1.42 times the larger element
  if (STYLE == DSR_ROPE_NEOX) {
    float y[8];
    mx_decode<FMT>(v.other, v.s_other, y);
    odd |= v.s_other >= top_scale<FMT, DT>();
    const bool lower = c < r.half_vecs;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float ps = y[e] * t[e >> 1][2 * (e & 1) + 1];
      x[e] = __builtin_fmaf(x[e], t[e >> 1][2 * (e & 1)], lower ? -ps : ps);
    }
  } else {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      const float cs = t[e >> 2][e & 2], sn = t[e >> 2][(e & 2) + 1];
      const float u = x[e], w = x[e + 1];
      const float us = u * sn, ws = w * sn;
      x[e] = __builtin_fmaf(u, cs, -ws);
      x[e + 1] = __builtin_fmaf(w, cs, us);
    }
  }
  return mx_store_vec<DT>(x, odd);
}

// The record vector that K's vector rv (column c of its row) turns with, or -1.
template <int STYLE>
__device__ __forceinline__ int mx_partner(const MxRope& r, int rv, int c) {
  if (STYLE != DSR_ROPE_NEOX || !r.rope_idx || c >= r.rot_vecs) return -1;
  return c < r.half_vecs ? rv + r.half_vecs : rv - r.half_vecs;
}
// K's vector, loaded with its partner, for table cs (null: not rotated).
template <int FMT, int DT, int STYLE>
__device__ __forceinline__ u32x4 mx_key_vec(const MxVec& v, int c, const MxRope& r,
                                            const float2* cs) {
  if (!cs || c >= r.rot_vecs) return mx_plain_vec<FMT, DT>(v);
  constexpr bool kNeox = STYLE == DSR_ROPE_NEOX;
  const int col = kNeox ? (c < r.half_vecs ? c : c - r.half_vecs) * 8 : c * 4;
  const f32x4* p = reinterpret_cast<const f32x4*>(cs + col);
  f32x4 t[4];
#pragma unroll
  for (int k = 0; k < (kNeox ? 4 : 2); ++k) t[k] = p[k];
  return mx_turned_vec<FMT, DT, STYLE>(v, c, r, t);
}

// Table of entry p in record layer l, or null.
__device__ __forceinline__ const float2* mx_table(const MxRope& r, int64_t p, int l) {
  if (!r.rope_idx) return nullptr;
  int t = r.rope_idx[p];
  if (t < 0 || t >= r.n_tables) return nullptr;
  if (r.layer_group) {
    const int g = r.layer_group[l];
    if (g < 0 || g >= r.n_groups) return nullptr;
    t += g * r.n_tables;
  }
  return r.cos_sin + (int64_t)t * (r.rot_vecs * 4);
}

struct MxPos {
  uint8_t* cache;
  uint8_t* rec;
  uint32_t page;
  int layer;  // of the record
  int part;
};

// This wave's piece, as flat_pos finds it; false past the launch's end and for entries
// out of bounds.
template <bool kPageMajor>
__device__ __forceinline__ bool mx_pos(const MxArgs& a, const FlatMap& m, const int32_t* page_ids,
                                       const int64_t* slot_offsets, MxPos* o) {
  const uint32_t w = flat_wave(m);
  if (w >= m.n_waves) return false;
  const uint32_t g = m.wave0 + w;
  const uint32_t q = div_by(g, m.per_unit);
  o->part = (int)(g - q * m.per_unit.d);
  const uint32_t v = m.unit0 + q;
  const uint32_t hi = div_by(v, m.minor);
  const uint32_t lo = v - hi * m.minor.d;
  const uint32_t p = kPageMajor ? hi : lo;
  const int l = a.first + (int)(kPageMajor ? lo : hi);
  const int64_t blk = page_ids[p];
  const int64_t rec = slot_offsets[p], off = rec + (int64_t)(a.layer0 + l) * a.layer_bytes;
  if (blk < 0 || blk >= a.num_blocks) return false;
  if (rec < 0 || off + a.need > a.staging_bytes) return false;
  o->cache = reinterpret_cast<uint8_t*>(a.layer_base[l]) + blk * a.page_stride;
  o->rec = a.staging + off;
  o->page = p;
  o->layer = a.layer0 + l;
  return true;
}

// Pages -> records. A wave takes 64 U vectors of K and of V in the record's order: rows of
// the cache page (256 bytes at head_dim 128) are read whole, codes and scales of U KiB of
// the cache go through the wave's LDS and are stored 16 bytes to a lane.
template <int FMT, int DT, bool HND, int U, int POLICY>
__global__ __launch_bounds__(kThreads) void kv_mx_gather_kernel(MxArgs a, const int32_t* page_ids,
                                                                const int64_t* slot_offsets,
                                                                FlatMap m) {
  constexpr int CB = mx_code_bytes<FMT>();
  __shared__ u32x4 lds[kThreads / kWave][(U * kWave * CB + U * 16) / 16];
  MxPos u;
  if (!mx_pos<true>(a, m, page_ids, slot_offsets, &u)) return;
  const int lane = (int)threadIdx.x % kWave;
  const int first = u.part * (kWave * U);
  const int left = a.vecs - first < kWave * U ? a.vecs - first : kWave * U;
  uint8_t* const mine = reinterpret_cast<uint8_t*>(lds[threadIdx.x / kWave]);
  u32x4 x[2][U];
#pragma unroll
  for (int k = 0; k < U; ++k) {
    const int rv = first + k * kWave + lane;
    int cv = rv;
    if (!HND) {
      const int row = (int)div_by((uint32_t)rv, a.row_vecs);
      const int c = rv - row * (int)a.row_vecs.d;
      const int h = (int)div_by((uint32_t)row, a.by_block);
      cv = ((row - h * a.block) * a.heads + h) * (int)a.row_vecs.d + c;
    }
    const int off = rv < a.vecs ? cv << 4 : (int)a.page_bytes;
#pragma unroll
    for (int half = 0; half < 2; ++half)
      x[half][k] = bload(make_rsrc(u.cache + (half ? a.kv_stride : 0), a.page_bytes), off);
  }
#pragma unroll
  for (int half = 0; half < 2; ++half) {
#pragma unroll
    for (int k = 0; k < U; ++k) {
      const uint32_t s = mx_scale_code<FMT>(mx_block_max<DT>(x[half][k]));
      const uint2 q = mx_encode<FMT, DT>(x[half][k], s);
      const int i = k * kWave + lane;
      if (FMT == DSR_MX_FP4) reinterpret_cast<uint32_t*>(mine)[i] = q.x;
      else reinterpret_cast<uint2*>(mine)[i] = q;
      if ((lane & 3) == 0) mine[U * kWave * CB + (i >> 2)] = (uint8_t)s;
    }
    wave_lds();
    const MxHalf o = mx_half(a, u.rec, half);
    const rsrc_t codes = make_rsrc(o.codes + (int64_t)first * CB, (int64_t)left * CB);
    const rsrc_t scales = make_rsrc(o.scales + first / 4, left / 4);
#pragma unroll
    for (int k = 0; k < (U * CB + 15) / 16; ++k) {
      const int i = k * kWave + lane;
      if (i * 16 < U * kWave * CB)
        bstore_as<POLICY>(codes, i * 16, reinterpret_cast<u32x4*>(mine)[i]);
    }
    if (lane < U * 16)
      __builtin_amdgcn_raw_buffer_store_b8(mine[U * kWave * CB + lane], scales, lane, 0, POLICY);
    wave_lds();  // before the other half's
  }
}

// Records -> pages. A wave takes 64 vectors of K and of V in the cache page's order.
template <int FMT, int DT, bool HND, int STYLE, int POLICY>
__global__ __launch_bounds__(kThreads) void kv_mx_scatter_kernel(MxArgs a, MxRope r,
                                                                 const int32_t* page_ids,
                                                                 const int64_t* slot_offsets,
                                                                 FlatMap m) {
  MxPos u;
  if (!mx_pos<false>(a, m, page_ids, slot_offsets, &u)) return;
  const int cv = u.part * kWave + (int)threadIdx.x % kWave;
  if (cv >= a.vecs) return;
  const int row = (int)div_by((uint32_t)cv, a.row_vecs);
  const int c = cv - row * (int)a.row_vecs.d;
  int rv = cv;
  if (!HND) {
    const int t = (int)div_by((uint32_t)row, a.by_heads);
    const int h = row - t * a.heads;
    rv = (h * a.block + t) * (int)a.row_vecs.d + c;
  }
  const rsrc_t ck = make_rsrc(u.cache, a.page_bytes);
  const rsrc_t cw = make_rsrc(u.cache + a.kv_stride, a.page_bytes);
  // the loads go out before the page's table is known
  const MxVec v = mx_load_vec<FMT>(mx_half(a, u.rec, 1), rv, -1);
  const MxVec w = mx_load_vec<FMT>(mx_half(a, u.rec, 0), rv, mx_partner<STYLE>(r, rv, c));
  const u32x4 k = mx_key_vec<FMT, DT, STYLE>(w, c, r, mx_table(r, u.page, u.layer));
  bstore_as<POLICY>(ck, cv << 4, k);
  bstore_as<POLICY>(cw, cv << 4, mx_plain_vec<FMT, DT>(v));
}

// The same where whole neox rows turn: a lane takes a vector of K and its partner, half a
// row on, so that each is decoded once and the table's entries are read once for both, and
// two vectors of V. Llama-3-8B from mxint8 (16.3 GB moved): 3.14 -> 2.98 ms at 5 workgroups
// a CU (4 2.98, 6 3.02, 8 3.08).
template <int FMT, int DT, bool HND, int POLICY>
__global__ __launch_bounds__(kThreads) void kv_mx_scatter_pairs_kernel(MxArgs a, MxRope r,
                                                                       const int32_t* page_ids,
                                                                       const int64_t* slot_offsets,
                                                                       FlatMap m, FastDiv by_half) {
  MxPos u;
  if (!mx_pos<false>(a, m, page_ids, slot_offsets, &u)) return;
  const int i = u.part * kWave + (int)threadIdx.x % kWave;  // pair, and two vectors of V
  if (2 * i >= a.vecs) return;
  const int nv = (int)a.row_vecs.d, hv = r.half_vecs;
  const int row = (int)div_by((uint32_t)i, by_half), c = i - row * hv;
  int rec_row = row;
  if (!HND) {
    const int t = (int)div_by((uint32_t)row, a.by_heads);
    rec_row = (row - t * a.heads) * a.block + t;
  }
  const MxHalf hk = mx_half(a, u.rec, 0), hw = mx_half(a, u.rec, 1);
  MxVec k, v[2];
  k = mx_load_vec<FMT>(hk, rec_row * nv + c, rec_row * nv + c + hv);
  v[0] = mx_load_vec<FMT>(hw, rec_row * nv + c, -1);
  v[1] = mx_load_vec<FMT>(hw, rec_row * nv + c + hv, -1);
  const float2* cs = mx_table(r, u.page, u.layer);
  const rsrc_t ck = make_rsrc(u.cache, a.page_bytes);
  const rsrc_t cw = make_rsrc(u.cache + a.kv_stride, a.page_bytes);
  const int off = (row * nv + c) << 4;
  u32x4 lower, upper;
  if (cs) {
    const f32x4* p = reinterpret_cast<const f32x4*>(cs + c * 8);
    f32x4 t[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) t[e] = p[e];
    float x[8], y[8], z[8];
    mx_decode<FMT>(k.own, k.s, x);
    mx_decode<FMT>(k.other, k.s_other, y);
    const bool odd = k.s >= top_scale<FMT, DT>() || k.s_other >= top_scale<FMT, DT>();
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const float cos = t[e >> 1][2 * (e & 1)], sin = t[e >> 1][2 * (e & 1) + 1];
      const float ys = y[e] * sin, xs = x[e] * sin;
      z[e] = __builtin_fmaf(y[e], cos, xs);
      x[e] = __builtin_fmaf(x[e], cos, -ys);
    }
    lower = mx_store_vec<DT>(x, odd);
    upper = mx_store_vec<DT>(z, odd);
  } else {
    lower = mx_plain_vec<FMT, DT>(k);
    upper = mx_plain_vec<FMT, DT>(MxVec{k.other, k.other, k.s_other, k.s_other});
  }
  bstore_as<POLICY>(ck, off, lower);
  bstore_as<POLICY>(ck, off + (hv << 4), upper);
  bstore_as<POLICY>(cw, off, mx_plain_vec<FMT, DT>(v[0]));
  bstore_as<POLICY>(cw, off + (hv << 4), mx_plain_vec<FMT, DT>(v[1]));
}

// The token form: lane = one vector of one token's K and V rows, layer blockIdx.y.
struct MxToken {
  uint8_t* cache;
  uint8_t* rec;
  int cv, rv, c;  // vectors in the cache page and in the record; column in the row
  int64_t token;
};
template <bool HND>
__device__ __forceinline__ bool mx_token(const MxArgs& a, const int64_t* slots,
                                         const int64_t* rows, uint32_t n, FastDiv per_token,
                                         int l, MxToken* o) {
  const uint32_t i = blockIdx.x * kThreads + threadIdx.x;
  const uint32_t t = div_by(i, per_token);
  if (t >= n) return false;
  const uint32_t v = i - t * per_token.d;
  const int h = (int)div_by(v, a.row_vecs);
  o->c = (int)(v - (uint32_t)h * a.row_vecs.d);
  const int64_t slot = slots[t], row = rows[t];
  if (slot < 0 || row < 0) return false;
  // a 64-bit division is some hundred instructions (67,000 tokens of Qwen2-0.5B loaded by
  // slot 289 -> 230 us, saved 277 -> 271)
  int64_t blk, off;
  if (a.block_shift >= 0) {
    blk = slot >> a.block_shift;
    off = row >> a.block_shift;
  } else {
    blk = slot / a.block;
    off = row / a.block;
  }
  const int ct = (int)(slot - blk * a.block), rt = (int)(row - off * a.block);
  if (blk >= a.num_blocks || (off & 15)) return false;
  const int64_t at = off + (int64_t)(a.layer0 + l) * a.layer_bytes;
  if (at + a.need > a.staging_bytes) return false;
  o->cache = reinterpret_cast<uint8_t*>(a.layer_base[l]) + blk * a.page_stride;
  o->rec = a.staging + at;
  o->cv = (HND ? h * a.block + ct : ct * a.heads + h) * (int)a.row_vecs.d + o->c;
  o->rv = (h * a.block + rt) * (int)a.row_vecs.d + o->c;
  o->token = t;
  return true;
}

template <int FMT, int DT, bool HND>
__global__ __launch_bounds__(kThreads) void kv_mx_gather_slots_kernel(MxArgs a,
                                                                      const int64_t* slots,
                                                                      const int64_t* rows,
                                                                      uint32_t n,
                                                                      FastDiv per_token) {
  MxToken u;
  // the 4 lanes of a block belong to one token and leave together
  if (!mx_token<HND>(a, slots, rows, n, per_token, a.first + (int)blockIdx.y, &u)) return;
#pragma unroll
  for (int half = 0; half < 2; ++half) {
    const u32x4 v = *reinterpret_cast<const u32x4*>(u.cache + (half ? a.kv_stride : 0) +
                                                    ((int64_t)u.cv << 4));
    const uint32_t s = mx_scale_code<FMT>(mx_block_max<DT>(v));
    const uint2 q = mx_encode<FMT, DT>(v, s);
    const MxHalf o = mx_half(a, u.rec, half);
    if (FMT == DSR_MX_FP4)
      reinterpret_cast<uint32_t*>(const_cast<uint8_t*>(o.codes))[u.rv] = q.x;
    else
      reinterpret_cast<uint2*>(const_cast<uint8_t*>(o.codes))[u.rv] = q;
    if ((u.rv & 3) == 0) const_cast<uint8_t*>(o.scales)[u.rv >> 2] = (uint8_t)s;
  }
}

template <int FMT, int DT, bool HND, int STYLE>
__global__ __launch_bounds__(kThreads) void kv_mx_scatter_slots_kernel(MxArgs a, MxRope r,
                                                                       const int64_t* slots,
                                                                       const int64_t* rows,
                                                                       uint32_t n,
                                                                       FastDiv per_token) {
  MxToken u;
  const int l = a.first + (int)blockIdx.y;
  if (!mx_token<HND>(a, slots, rows, n, per_token, l, &u)) return;
  const float2* cs = mx_table(r, u.token, a.layer0 + l);
  const MxVec x = mx_load_vec<FMT>(mx_half(a, u.rec, 1), u.rv, -1);
  const MxVec w = mx_load_vec<FMT>(mx_half(a, u.rec, 0), u.rv, mx_partner<STYLE>(r, u.rv, u.c));
  const u32x4 v = mx_plain_vec<FMT, DT>(x);
  const u32x4 k = mx_key_vec<FMT, DT, STYLE>(w, u.c, r, cs);
  *reinterpret_cast<u32x4*>(u.cache + ((int64_t)u.cv << 4)) = k;
  *reinterpret_cast<u32x4*>(u.cache + a.kv_stride + ((int64_t)u.cv << 4)) = v;
}

}  // namespace
