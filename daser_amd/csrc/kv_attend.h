// kv_attend.h -- attention over quantised records.
// Part of libdaser_kv: included by kv_mx.hip.
//
// out = sum_t p_t v_t, p = softmax(scale q . R(d) k_t): the records' rows are read
// in place. A moved chunk's keys R(d) k meet the queries as q . R(d) k = (R(-d) q) . k,
// so the query is rotated, once per chunk, and the keys are not.
//
// One wave per (query row, head): 64 tokens at a time, each lane one token's score,
// then each lane D / 64 columns of the values.

#pragma once

#include "kv_mx.h"

namespace {

struct AttendArgs {
  dsr_attend_args a;
  int32_t codes, scales;  // section bytes of one half
  int64_t need;
};

template <int FMT>
__device__ __forceinline__ float mx_element(const uint8_t* codes, const uint8_t* scales,
                                            int64_t i) {
  const uint32_t s = scales[i >> 5];
  if (s == 255u) return __uint_as_float(0x7fc00000u);
  if (FMT == DSR_MX_INT8) return __builtin_ldexpf((float)(int8_t)codes[i], (int)s - 133);
  const uint32_t c = codes[i >> 1] >> (4 * (i & 1)) & 15u;
  const uint32_t e = c >> 1 & 3u, f = c & 1u;
  const float m = e ? __builtin_ldexpf(1.0f + 0.5f * f, (int)e - 1) : 0.5f * f;
  return __builtin_ldexpf(c & 8u ? -m : m, (int)s - 127);
}

template <int DT>
__device__ __forceinline__ float read16(const void* p, int64_t i) {
  const uint32_t h = static_cast<const uint16_t*>(p)[i];
  return DT == DSR_DTYPE_BF16 ? bf16_to_f32(h) : fp16_to_f32(h);
}
template <int DT>
__device__ __forceinline__ float as_type(float f) {  // as a cache of the type holds it
  const float top = DT == DSR_DTYPE_BF16 ? __uint_as_float(0x7f7f0000u) : 65504.0f;
  f = f > top ? top : f;
  f = f < -top ? -top : f;
  return DT == DSR_DTYPE_BF16 ? bf16_to_f32(f32_to_bf16(f)) : fp16_to_f32(f32_to_fp16(f));
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

template <int FMT, int DT>
__global__ __launch_bounds__(kWave) void kv_mx_attend_simple_kernel(AttendArgs g) {
  const dsr_attend_args& a = g.a;
  const int lane = (int)threadIdx.x, hq = (int)blockIdx.y, r = (int)blockIdx.z;
  const int D = a.head_dim, bs = a.block_size;
  const int h = hq / (a.q_heads / a.kv_heads);
  __shared__ float qs[256], ps[kWave];
  const int q0 = clampi(a.q_start[r], 0, a.n_q), q1 = clampi(a.q_start[r + 1], 0, a.n_q);
  const int p0 = clampi(a.page_start[r], 0, a.n_pages);
  const int p1 = clampi(a.page_start[r + 1], p0, a.n_pages);
  const float ninf = -__builtin_inff();
  for (int i = q0 + (int)blockIdx.x; i < q1; i += (int)gridDim.x) {
    int64_t ctx = a.context[r];
    if (a.limits && a.limits[i] < ctx) ctx = a.limits[i];
    if (ctx > (int64_t)(p1 - p0) * bs) ctx = (int64_t)(p1 - p0) * bs;
    const uint8_t* q = static_cast<const uint8_t*>(a.q) + (int64_t)i * a.q_row_stride +
                       (int64_t)hq * a.q_head_stride;
    float m = ninf, sum = 0.0f, acc[4] = {0, 0, 0, 0};
    int table = -2;
    for (int64_t t0 = 0; t0 < ctx; t0 += bs) {  // a page at a time
      const int p = p0 + (int)(t0 / bs);
      const int64_t at = a.slot_offsets[p], off = at + (int64_t)a.layer * a.layer_bytes;
      if (at < 0 || (off & 15) || off + g.need > a.staging_bytes) continue;
      const uint8_t* rec = static_cast<const uint8_t*>(a.staging) + off;
      int ti = a.rope_idx ? a.rope_idx[p] : -1;
      if (ti >= a.n_tables) ti = -1;
      if (ti != table) {
        __syncthreads();
        const float2* cs = reinterpret_cast<const float2*>(a.cos_sin) + (int64_t)ti * (a.rot_dim / 2);
        for (int d = lane; d < D; d += kWave) {
          float x = read16<DT>(q, d);
          if (ti >= 0 && d < a.rot_dim) {
            const int half = a.rot_dim / 2;
            const bool neox = a.style == DSR_ROPE_NEOX;
            const bool lower = neox ? d < half : (d & 1) == 0;
            const float y = read16<DT>(q, neox ? (lower ? d + half : d - half) : d ^ 1);
            const float2 w = cs[neox ? (lower ? d : d - half) : d >> 1];
            x = x * w.x + (lower ? y * w.y : -(y * w.y));  // by -delta
          }
          qs[d] = x;
        }
        table = ti;
        __syncthreads();
      }
      const uint8_t* vc = rec + g.codes;
      const uint8_t* ks = rec + 2 * (int64_t)g.codes;
      const uint8_t* vs = ks + g.scales;
      for (int b = 0; b < bs && t0 + b < ctx; b += kWave) {
        const int n = bs - b < kWave ? bs - b : kWave;
        const bool seen = lane < n && t0 + b + lane < ctx;
        float s = ninf;
        if (seen) {
          s = 0.0f;
          const int64_t row = ((int64_t)h * bs + b + lane) * D;
          for (int d = 0; d < D; ++d) s += qs[d] * as_type<DT>(mx_element<FMT>(rec, ks, row + d));
          s *= a.scale;
        }
        float top = s;
        for (int k = 32; k; k >>= 1) {
          const float o = __shfl_xor(top, k);
          top = top > o || __builtin_isnan(top) ? top : o;  // a NaN stays
        }
        const float mn = m > top || __builtin_isnan(m) ? m : top;
        const float keep = m == ninf ? 0.0f : __expf(m - mn);
        const float pr = seen ? __expf(s - mn) : 0.0f;
        float part = pr;
        for (int k = 32; k; k >>= 1) part += __shfl_xor(part, k);
        sum = sum * keep + part;
        m = mn;
        __syncthreads();
        ps[lane] = pr;
        __syncthreads();
        for (int j = 0; j * kWave < D; ++j) {
          const int d = j * kWave + lane;
          acc[j] *= keep;
          if (d >= D) continue;
          for (int t = 0; t < n && t0 + b + t < ctx; ++t)
            acc[j] += ps[t] * as_type<DT>(mx_element<FMT>(vc, vs, ((int64_t)h * bs + b + t) * D + d));
        }
      }
    }
    float lse = m == ninf ? ninf : m + __logf(sum);
    float own = sum > 0.0f || __builtin_isnan(sum) ? 1.0f / sum : 0.0f, other = 0.0f;
    const int64_t at = (int64_t)i * a.q_heads + hq;
    if (a.prior_out) {
      const float l2 = a.prior_lse[at], top = l2 > lse ? l2 : lse;
      if (top != ninf) {
        const float e1 = __expf(lse - top), e2 = __expf(l2 - top);
        own *= e1 / (e1 + e2);
        other = e2 / (e1 + e2);
        lse = top + __logf(e1 + e2);
      }
    }
    for (int j = 0; j * kWave < D; ++j) {
      const int d = j * kWave + lane;
      if (d >= D) continue;
      float o = acc[j] * own;
      if (other != 0.0f) o += other * read16<DT>(a.prior_out, at * D + d);
      static_cast<uint16_t*>(a.out)[at * D + d] =
          (uint16_t)(DT == DSR_DTYPE_BF16 ? f32_to_bf16(o) : f32_to_fp16(o));
    }
    if (lane == 0) a.lse[at] = lse;
  }
}

}  // namespace
