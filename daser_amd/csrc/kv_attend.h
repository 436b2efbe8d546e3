// kv_attend.h -- attention over quantised records.
// Part of libdaser_kv: included by kv_attend.hip.
//
// out = sum_t p_t v_t, p = softmax(scale q . R(d) k_t): the records' rows are read
// in place. A moved chunk's keys R(d) k meet the queries as q . R(d) k = (R(-d) q) . k,
// so the query is rotated, once per chunk, and the keys are not.
//
// A workgroup takes one request, one KV head, a tile of 16 NQ query rows (query tokens
// times the heads that share the KV head) and a stretch of the tokens; its 4 waves take
// turns at steps of 32 tokens. Per step and wave:
//   S^T = K Q^T    tokens x rows, so that a lane holds 4 consecutive tokens of one row.
//                  Lane (n, g) dequantises the quarter g of row n, one 16-byte load of
//                  e2m1 at head_dim 128, and the MFMA's k index runs over the quarters.
//   P              exponentials against a running maximum that is renewed only when a
//                  score passes it by 2^8, so that the usual step has no reduction.
//   O^T += V^T P^T P^T is in the MFMA's operand layout as it comes from S^T. V is
//                  dequantised to LDS row by row and read back transposed
//                  (ds_read_b64_tr_b16); the wave uses its own part, without barriers.
// K and V are exact in q's type, products and sums are fp32, P is rounded to q's type.

#pragma once

#include "kv_mx.h"

namespace {

struct AttendArgs {
  dsr_attend_args a;
  int32_t codes, scales;  // section bytes of one half
  int64_t need;
  int32_t group;          // query heads per KV head
  int32_t tiles, splits;  // of blockIdx.x
  int32_t chunk;          // tokens of a split (the last one takes the rest)
  int32_t wave_heads;     // KV heads of a workgroup: 4 / wave_heads waves share a head's tokens
  float scale2;           // scale * log2(e)
  FastDiv by_block;       // tokens to pages
  float* part_o;          // [n_q * q_heads][splits][head_dim]
  float2* part_ml;        // [n_q * q_heads][splits] (maximum in log2 units, sum)
};

template <int DT>
__device__ __forceinline__ float read16(const void* p, int64_t i) {
  const uint32_t h = static_cast<const uint16_t*>(p)[i];
  return DT == DSR_DTYPE_BF16 ? bf16_to_f32(h) : fp16_to_f32(h);
}

__device__ __forceinline__ int clampi(int x, int lo, int hi) {
  return x < lo ? lo : x > hi ? hi : x;
}

constexpr int kMaxTokens = 0x7fff0000;  // of a request, that 32 more are an int too

// Request r: its query rows [q0, q1), its pages from p0, its tokens.
struct AttendRequest {
  int q0, q1, p0, p1;
  int64_t tokens;
};
__device__ __forceinline__ AttendRequest attend_request(const dsr_attend_args& a, int r) {
  AttendRequest o;
  o.q0 = clampi(a.q_start[r], 0, a.n_q);
  o.q1 = clampi(a.q_start[r + 1], 0, a.n_q);
  o.p0 = clampi(a.page_start[r], 0, a.n_pages);
  o.p1 = clampi(a.page_start[r + 1], o.p0, a.n_pages);
  const int64_t held = (int64_t)(o.p1 - o.p0) * a.block_size;
  o.tokens = a.context[r];
  o.tokens = o.tokens < 0 ? 0 : o.tokens > held ? held : o.tokens;
  if (o.tokens > kMaxTokens) o.tokens = kMaxTokens;
  return o;
}

// 2^x; log2.
__device__ __forceinline__ float exp2_(float x) { return __builtin_amdgcn_exp2f(x); }
__device__ __forceinline__ float log2_(float x) { return __builtin_amdgcn_logf(x); }
constexpr float kLn2 = 0.69314718055994531f;

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef short s16x4 __attribute__((ext_vector_type(4)));

template <int DT>
__device__ __forceinline__ f32x4 mfma32(u32x4 a, u32x4 b, f32x4 c) {
  if constexpr (DT == DSR_DTYPE_BF16)
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a),
                                                   __builtin_bit_cast(bf16x8, b), c, 0, 0, 0);
  else
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, a),
                                                  __builtin_bit_cast(f16x8, b), c, 0, 0, 0);
}

template <int DT>
__device__ __forceinline__ float half_of(uint32_t w, int k) {
  const uint32_t h = k ? w >> 16 : w & 0xffffu;
  return DT == DSR_DTYPE_BF16 ? bf16_to_f32(h) : fp16_to_f32(h);
}

// out[i][h] and its lse from the unnormalised sum o (4 consecutive columns from d on),
// the maximum m (log2 units) and the sum l of this kernel's part, and the prior's.
struct AttendScale {
  float own, other, lse;
};
__device__ __forceinline__ AttendScale attend_scale(const dsr_attend_args& a, int64_t at, float m,
                                                    float l) {
  const float ninf = -__builtin_inff();
  AttendScale o;
  o.lse = l == 0.0f ? ninf : (m + log2_(l)) * kLn2;
  o.own = l == 0.0f ? 0.0f : 1.0f / l;
  o.other = 0.0f;
  if (a.prior_out) {
    const float l2 = a.prior_lse[at];
    const float top = l2 > o.lse ? l2 : o.lse;
    if (top != ninf) {
      const float e1 = exp2_((o.lse - top) / kLn2), e2 = exp2_((l2 - top) / kLn2);
      o.own *= e1 / (e1 + e2);
      o.other = e2 / (e1 + e2);
      o.lse = top + log2_(e1 + e2) * kLn2;
    }
  }
  return o;
}
template <int DT>
__device__ __forceinline__ void attend_store(const dsr_attend_args& a, int64_t at, int d, f32x4 o,
                                             const AttendScale& s) {
  const int64_t i = at * a.head_dim + d;
#pragma unroll
  for (int k = 0; k < 4; ++k) {
    o[k] = s.own == 0.0f ? 0.0f : o[k] * s.own;
    if (s.other != 0.0f) o[k] += s.other * read16<DT>(a.prior_out, i + k);
  }
  uint2 w{pack2<DT>(o[0], o[1]), pack2<DT>(o[2], o[3])};
  *reinterpret_cast<uint2*>(static_cast<uint16_t*>(a.out) + i) = w;
}

// One 16-token tile as loaded: this lane's quarter of K row and V row n, and their scales.
template <int FMT, int D>
struct AttendTile {
  static constexpr int W = (FMT == DSR_MX_FP4 ? 1 : 2) * (D / 32);  // dwords of a quarter
  static constexpr int S = D == 96 || D == 256 ? 2 : 1;             // blocks it touches
  uint32_t k[W], v[W];
  uint32_t ks[S], vs[S];
};

template <int W, int POLICY>
__device__ __forceinline__ void load_words(rsrc_t r, int off, uint32_t* w) {
  typedef unsigned int u32x2 __attribute__((ext_vector_type(2)));
  typedef unsigned int u32x3 __attribute__((ext_vector_type(3)));
  int i = 0;
  if constexpr (W >= 4) {
#pragma unroll
    for (int k = 0; k < W / 4; ++k, i += 4) {
      const u32x4 x = __builtin_amdgcn_raw_buffer_load_b128(r, off + 16 * k, 0, POLICY);
      w[i] = x[0];
      w[i + 1] = x[1];
      w[i + 2] = x[2];
      w[i + 3] = x[3];
    }
  }
  constexpr int rest = W % 4, at = W / 4 * 4;
  if constexpr (rest == 1) w[at] = __builtin_amdgcn_raw_buffer_load_b32(r, off + 4 * at, 0, POLICY);
  if constexpr (rest == 2) {
    const u32x2 x = __builtin_amdgcn_raw_buffer_load_b64(r, off + 4 * at, 0, POLICY);
    w[at] = x[0];
    w[at + 1] = x[1];
  }
  if constexpr (rest == 3) {
    const u32x3 x = __builtin_amdgcn_raw_buffer_load_b96(r, off + 4 * at, 0, POLICY);
    w[at] = x[0];
    w[at + 1] = x[1];
    w[at + 2] = x[2];
  }
}

// Entries of 64 pages, one to a lane: the offset of the page's layer (-1: not there, or
// outside the records) and its table.
struct AttendPages {
  int64_t off;
  int table;
};
struct AttendPage {
  int64_t off;
  int table;
};
template <bool ROPE>
__device__ __forceinline__ AttendPages attend_pages(const AttendArgs& g, const AttendRequest& rq,
                                                    int page, int lane) {
  const dsr_attend_args& a = g.a;
  AttendPages o{-1, -1};
  const int64_t p = (int64_t)rq.p0 + page + lane;
  if (p < rq.p1) {
    const int64_t at = a.slot_offsets[p], off = at + (int64_t)a.layer * a.layer_bytes;
    if (at >= 0 && (at & 15) == 0 && off + g.need <= a.staging_bytes) o.off = off;
    if (ROPE) {
      o.table = a.rope_idx[p];
      if (o.table < -1 || o.table >= a.n_tables) o.table = -1;
    }
  }
  return o;
}
template <bool ROPE>
__device__ __forceinline__ AttendPage page_of(const AttendPages& x, int i) {
  const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x.off, i);
  const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(x.off >> 32), i);
  return {(int64_t)((uint64_t)hi << 32 | lo), ROPE ? __builtin_amdgcn_readlane(x.table, i) : -1};
}

// Query rows of this lane's columns as MFMA operands: chunk i of its quarter. Rows that do
// not exist (bit j of `in` clear) point to one that does and become zeros: without branches
// the loads go out together.
template <int D, int NQ>
__device__ __forceinline__ void load_queries(const uint8_t* const* rows, uint32_t in, int quarter,
                                             u32x4 (*hi)[D / 32]) {
  constexpr int B = D / 32;
#pragma unroll
  for (int j = 0; j < NQ; ++j) {
    const uint32_t mask = in >> j & 1 ? ~0u : 0u;
#pragma unroll
    for (int i = 0; i < B; ++i)
      hi[j][i] = *reinterpret_cast<const u32x4*>(rows[j] + 16 * (quarter * B + i)) & mask;
  }
}
// One of those rows rotated by -delta with table cs; lo: what the rounding of hi left. The
// chunks are made in a loop that stays one and pass through `room` (2 KiB a chunk of the
// wave's LDS, free between steps): unrolled, their values push the accumulators out of the
// registers (questions over moved chunks 98 -> 133 us).
template <int DT, int D>
__device__ __forceinline__ void turn_query(const dsr_attend_args& a, const uint8_t* row, bool in,
                                           int quarter, const float2* cs, char* room, u32x4* hi,
                                           u32x4* lo) {
  constexpr int B = D / 32;
  const bool neox = a.style == DSR_ROPE_NEOX;
  const int half = a.rot_dim / 16;  // chunks to the neox partner
  const uint32_t mask = in ? ~0u : 0u;
  char* const put = room + (int)(threadIdx.x % kWave) * 16;
#pragma unroll 1
  for (int i = 0; i < B; ++i) {
    const int c = quarter * B + i;  // 8 elements
    const bool turned = c * 8 < a.rot_dim;
    const bool lower = c < half;
    const int pair = !turned ? 0 : neox ? (lower ? c : c - half) * 8 : c * 4;
    const int partner = !turned || !neox ? c : lower ? c + half : c - half;
    const f32x4* p = reinterpret_cast<const f32x4*>(cs + pair);
    // two pairs each: 8 (neox) or 4 (gptj, whose second half is not used) of them
    const f32x4 t[4] = {p[0], p[1], p[neox ? 2 : 0], p[neox ? 3 : 1]};
    const float flip = neox && !lower ? -1.0f : 1.0f;
    const u32x4 x = *reinterpret_cast<const u32x4*>(row + 16 * c) & mask;
    const u32x4 y = *reinterpret_cast<const u32x4*>(row + 16 * partner) & mask;
    u32x4 h, l;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
      const float x0 = half_of<DT>(x[k], 0), x1 = half_of<DT>(x[k], 1);
      // neox: pairs (2 k, 2 k + 1) with the partner's; gptj: pair k with itself
      const float y0 = neox ? half_of<DT>(y[k], 0) : x1, y1 = neox ? half_of<DT>(y[k], 1) : -x0;
      const float c0 = neox ? t[k][0] : t[k >> 1][2 * (k & 1)];
      const float s0 = neox ? t[k][1] : t[k >> 1][2 * (k & 1) + 1];
      const float c1 = neox ? t[k][2] : c0, s1 = neox ? t[k][3] : s0;
      const float r0 = turned ? x0 * c0 + y0 * (flip * s0) : x0;
      const float r1 = turned ? x1 * c1 + y1 * (flip * s1) : x1;
      h[k] = pack2<DT>(r0, r1);
      l[k] = pack2<DT>(r0 - half_of<DT>(h[k], 0), r1 - half_of<DT>(h[k], 1));
    }
    *reinterpret_cast<u32x4*>(put + i * 2048) = h;
    *reinterpret_cast<u32x4*>(put + i * 2048 + 1024) = l;
  }
#pragma unroll
  for (int i = 0; i < B; ++i) {
    hi[i] = *reinterpret_cast<const u32x4*>(put + i * 2048);
    lo[i] = *reinterpret_cast<const u32x4*>(put + i * 2048 + 1024);
  }
}

// The scheduler moves nothing past it: what it would fetch early costs registers.
__device__ __forceinline__ void phase() { __builtin_amdgcn_sched_barrier(0); }

constexpr int kAttendWaves = 4;
constexpr int kStep = 32;  // tokens of a step

// Bytes of a V row in LDS: 32 more than it holds, so that 8 rows of two 16-byte chunks (a
// transposing read of 32 lanes) and 8 rows of one (a write of 8 lanes) meet each bank once,
// and every address is a lane's base and a constant.
template <int D>
__device__ __forceinline__ constexpr int lds_row() {
  return 2 * D + 32;
}

// Waves per SIMD that the registers are to leave room for. Decode batch (e2m1, head_dim
// 128) at 2, 3 and 4: 174, 177 and 179 us before the grid was made odd; a moved chunk's
// queries spill 20 to 40 registers at 3, beside 2 waves' 106 us for questions (98 and 83
// with fewer spills). What bounds the decode batch is its 1 KiB reads, 131 us by themselves.
template <int D, int NQ, bool ROPE>
constexpr int attend_waves() {
  if (NQ == 1) return D <= 64 ? 4 : D <= 128 ? 3 : 2;
  return D * NQ <= 256 ? 2 : 1;
}

template <int FMT, int DT, int D, int NQ, bool ROPE>
__global__ __launch_bounds__(kThreads, (attend_waves<D, NQ, ROPE>())) void kv_mx_attend_kernel(
    AttendArgs g) {
  const dsr_attend_args& a = g.a;
  constexpr int B = D / 32, NT = D / 16;
  using Tile = AttendTile<FMT, D>;
  __shared__ u32x4 lds[kAttendWaves * kStep * lds_row<D>() / 16];
  __shared__ float2 lds_ml[kAttendWaves][16];
  const int lane = (int)threadIdx.x % kWave;
  const int wave = __builtin_amdgcn_readfirstlane((int)threadIdx.x / kWave);
  const int n = lane & 15, quarter = lane >> 4;
  char* const mine = reinterpret_cast<char*>(lds) + wave * kStep * lds_row<D>();
  char* const put = mine + n * lds_row<D>() + quarter * (16 * B);
  char* const get = mine + (4 * quarter + (n >> 2)) * lds_row<D>() + (n & 3) * 8;
  const int h = (int)blockIdx.y * g.wave_heads + wave % g.wave_heads;
  const int share = kAttendWaves / g.wave_heads;  // waves of a head
  const int split = (int)blockIdx.x % g.splits, tile0 = (int)blockIdx.x / g.splits;
  if (tile0 >= g.tiles) return;  // the odd one of the grid
  const AttendRequest rq = attend_request(a, (int)blockIdx.z);
  const int64_t rows = rq.q1 > rq.q0 ? (int64_t)(rq.q1 - rq.q0) * g.group : 0;
  const float ninf = -__builtin_inff();
  auto out_row = [&](int64_t row, int head) {
    return (int64_t)(rq.q0 + (int)(row / g.group)) * a.q_heads + head * g.group +
           (int)(row % g.group);
  };

  for (int64_t row0 = (int64_t)tile0 * (16 * NQ); row0 < rows;
       row0 += (int64_t)g.tiles * (16 * NQ)) {
    // this lane's columns
    int lim[NQ];
    const uint8_t* qrow[NQ];
    uint32_t in = 0;  // bit j: the column's row exists
    int tmax = 0, tmin = 0x7fffffff;
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      const int64_t row = row0 + 16 * j + n < rows ? row0 + 16 * j + n : rows - 1;
      const bool is = row0 + 16 * j + n < rows;
      const int i = rq.q0 + (int)((uint32_t)row / (uint32_t)g.group);
      const int hq = (int)((uint32_t)row % (uint32_t)g.group);
      int64_t seen = rq.tokens;
      if (a.limits && a.limits[i] < seen) seen = a.limits[i];
      lim[j] = !is || seen < 0 ? 0 : (int)seen;
      if (is && lim[j] < tmin) tmin = lim[j];
      if (lim[j] > tmax) tmax = lim[j];
      in |= (uint32_t)is << j;
      qrow[j] = static_cast<const uint8_t*>(a.q) + (int64_t)i * a.q_row_stride +
                (int64_t)(h * g.group + hq) * a.q_head_stride;
    }
#pragma unroll
    for (int k = 1; k < 16; k <<= 1) {
      const int x = __shfl_xor(tmax, k), y = __shfl_xor(tmin, k);
      tmax = x > tmax ? x : tmax;
      tmin = y < tmin ? y : tmin;
    }
    tmax = __builtin_amdgcn_readfirstlane(tmax);
    tmin = __builtin_amdgcn_readfirstlane(tmin);
    const int64_t begin64 = (int64_t)split * g.chunk;
    const int begin = begin64 < tmax ? (int)begin64 : tmax;
    int end = tmax;
    if (split < g.splits - 1 && tmax - begin > g.chunk) end = begin + g.chunk;
    if (begin >= end && split > 0) continue;  // the join does not read it

    u32x4 qh[NQ][B], ql[ROPE ? NQ : 1][ROPE ? B : 1];
    load_queries<D, NQ>(qrow, in, quarter, qh);
    if constexpr (ROPE)
#pragma unroll
      for (int j = 0; j < NQ; ++j)
#pragma unroll
        for (int i = 0; i < B; ++i) ql[j][i] = u32x4{0u, 0u, 0u, 0u};
    f32x4 acc[NQ][NT];
    float m[NQ], l[NQ];
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      m[j] = ninf;
      l[j] = 0.0f;
#pragma unroll
      for (int t = 0; t < NT; ++t) acc[j][t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }

    // This wave's tokens: its share of the stretch. The page tables' entries of 64 pages
    // lie in the lanes, those of the next 64 are under way.
    const int per = ((end - begin + share - 1) / share + kStep - 1) / kStep * kStep;
    const int turn = wave / g.wave_heads;
    const int first = end - begin > turn * per ? begin + turn * per : end;
    const int last = end - first > per ? first + per : end;
    int page0 = (int)div_by((uint32_t)first, g.by_block);
    AttendPages pages = attend_pages<ROPE>(g, rq, page0, lane);
    AttendPages later = attend_pages<ROPE>(g, rq, page0 + kWave, lane);
    // The step whose loads are under way: its tiles, which of them count, its first token, its
    // table. (Two steps ahead cost the registers of a third wave: decode batch 174 -> 198 us.)
    Tile tile[2];
    bool seen[2];
    int at, turned;
    int next = first;
    // the step at t: one tile only where the next one is moved otherwise, or its page's
    // entry is not in the lanes yet
    auto load_step = [&]() {
      const int t = next;
      at = t;
      if (t >= last) return;
      if ((int)div_by((uint32_t)t, g.by_block) - page0 >= kWave) {
        page0 += kWave;
        pages = later;
        later = attend_pages<ROPE>(g, rq, page0 + kWave, lane);
      }
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const int tt = t + 16 * u;
        const int p = (int)div_by((uint32_t)tt, g.by_block);
        const AttendPage e = page_of<ROPE>(pages, (p - page0) & (kWave - 1));
        seen[u] = tt < last && e.off >= 0;
        if (u == 0) {
          turned = e.table;
          next = t + kStep;
        } else if (p - page0 >= kWave || (ROPE && e.table != turned)) {
          seen[1] = false;
          next = t + 16;
        }
        const rsrc_t r = make_rsrc(static_cast<const uint8_t*>(a.staging) + (seen[u] ? e.off : 0),
                                   seen[u] ? g.need : 0);
        const int row = h * a.block_size + (tt - p * a.block_size) + n;
        const int at_k = row * (Tile::W * 16) + quarter * (Tile::W * 4);
        // one tile of rows reads them once: they stream through
        constexpr int kPolicy = NQ == 1 ? kLoadPolicy : 0;
        load_words<Tile::W, kPolicy>(r, at_k, tile[u].k);
        load_words<Tile::W, kPolicy>(r, at_k + g.codes, tile[u].v);
        const int at_s = 2 * g.codes + row * B;
        const int b0 = B * quarter / 4, b1 = (B * quarter + B - 1) / 4;
        tile[u].ks[0] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, at_s + b0, 0, 0);
        tile[u].vs[0] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, at_s + g.scales + b0, 0, 0);
        if constexpr (Tile::S == 2) {
          tile[u].ks[1] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, at_s + b1, 0, 0);
          tile[u].vs[1] = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, at_s + g.scales + b1, 0, 0);
        }
      }
    };
    // the scale of chunk i of this lane's quarter
    auto scale_of = [&](const uint32_t* s, int i) -> uint32_t {
      if constexpr (Tile::S == 1) return s[0];
      return (B * quarter + i) / 4 == B * quarter / 4 ? s[0] : s[1];
    };
    // One step on the loaded tiles. odd: scales near the type's largest value or NaN;
    // masked: tokens that some query does not see, or a tile missing. Both are rare and the
    // same for the wave.
    int held = -1;  // the table that the queries are rotated by
    auto run_step = [&]() {
      const int t0 = at;
      const bool now[2] = {seen[0], seen[1]};
      if constexpr (ROPE) {
        if (turned != held) {
          held = turned;
          if (held >= 0) {
            const float2* cs =
                reinterpret_cast<const float2*>(a.cos_sin) + (int64_t)held * (a.rot_dim / 2);
#pragma unroll
            for (int j = 0; j < NQ; ++j) {
              turn_query<DT, D>(a, qrow[j], in >> j & 1, quarter, cs, mine, qh[j], ql[j]);
              phase();
            }
          } else {
            load_queries<D, NQ>(qrow, in, quarter, qh);
#pragma unroll
            for (int j = 0; j < NQ; ++j)
#pragma unroll
              for (int i = 0; i < B; ++i) ql[j][i] = u32x4{0u, 0u, 0u, 0u};
          }
        }
      }
      bool odd = false;
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int i = 0; i < Tile::S; ++i)
          odd |= tile[u].ks[i] > top_scale<FMT, DT>() || tile[u].vs[i] > top_scale<FMT, DT>();
      odd = __any(odd);
      const bool masked = t0 + kStep > tmin || !now[0] || !now[1];
      f32x4 s[NQ][2];
      uint32_t nan_scale[2][Tile::S];
      // S of each tile; V to LDS, its NaN blocks as zeros that are put back below
#pragma unroll
      for (int u = 0; u < 2; ++u) {
        const bool row_in = now[u] && t0 + 16 * u + n < tmax;
        u32x4 vf[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
          vf[i] = dequantise<FMT, DT>(tile[u].v + i * (Tile::W / B), scale_of(tile[u].vs, i));
        if (__builtin_expect(odd, 0)) {
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const uint32_t sv = scale_of(tile[u].vs, i);
            if (sv > top_scale<FMT, DT>())
              vf[i] = dequantise_any<FMT, DT>(tile[u].v + i * (Tile::W / B), sv);
            if (sv == 255u || !row_in) vf[i] = u32x4{0u, 0u, 0u, 0u};
          }
        }
#pragma unroll
        for (int i = 0; i < B; ++i)
          *reinterpret_cast<u32x4*>(put + u * (16 * lds_row<D>()) + 16 * i) = vf[i];
        phase();
        u32x4 kf[B];
#pragma unroll
        for (int i = 0; i < B; ++i)
          kf[i] = dequantise<FMT, DT>(tile[u].k + i * (Tile::W / B), scale_of(tile[u].ks, i));
        if (__builtin_expect(odd, 0)) {
#pragma unroll
          for (int i = 0; i < B; ++i) {
            const uint32_t sk = scale_of(tile[u].ks, i);
            if (sk > top_scale<FMT, DT>())
              kf[i] = dequantise_any<FMT, DT>(tile[u].k + i * (Tile::W / B), sk);
          }
        }
#pragma unroll
        for (int j = 0; j < NQ; ++j) {
          s[j][u] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
          for (int i = 0; i < B; ++i) {
            s[j][u] = mfma32<DT>(kf[i], qh[j][i], s[j][u]);
            if (ROPE) s[j][u] = mfma32<DT>(kf[i], ql[j][i], s[j][u]);
          }
        }
#pragma unroll
        for (int i = 0; i < Tile::S; ++i) nan_scale[u][i] = tile[u].vs[i];
        phase();
      }
      load_step();
      phase();

      // P
      u32x4 pf[NQ];
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        float x[8];
        const float base = m[j] == ninf ? 0.0f : m[j];
        float top = ninf;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = __builtin_fmaf(s[j][e >> 2][e & 3], g.scale2, -base);
        }
        if (__builtin_expect(masked, 0)) {
#pragma unroll
          for (int e = 0; e < 8; ++e)
            if (t0 + 16 * (e >> 2) + 4 * quarter + (e & 3) >= lim[j] || !now[e >> 2]) x[e] = ninf;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) top = __builtin_fmaxf(top, x[e]);
        if (__any(top > 8.0f || (m[j] == ninf && top > ninf))) {
          top = __builtin_fmaxf(top, __shfl_xor(top, 16));
          top = __builtin_fmaxf(top, __shfl_xor(top, 32));
          const float mn = __builtin_fmaxf(m[j], top + base);
          if (mn != ninf) {
            const float keep = exp2_(m[j] - mn);
            const float shift = mn - base;
            m[j] = mn;
            l[j] *= keep;
#pragma unroll
            for (int k = 0; k < NT; ++k) acc[j][k] *= keep;
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] -= shift;
          }
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          x[e] = exp2_(x[e]);
          l[j] += x[e];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) pf[j][k] = pack2<DT>(x[2 * k], x[2 * k + 1]);
        phase();
      }

      wave_lds();
      // O^T: lanes' columns 4 c ... of rows 4 quarter + r, transposed in 16-lane groups
#pragma unroll
      for (int k = 0; k < NT; ++k) {
        union {
          s16x4 h[2];
          u32x4 v;
        } vt;
#pragma unroll
        for (int u = 0; u < 2; ++u)
          vt.h[u] = __builtin_amdgcn_ds_read_tr16_b64_v4i16(
              (__attribute__((address_space(3))) s16x4*)(get + u * (16 * lds_row<D>()) + 32 * k));
#pragma unroll
        for (int j = 0; j < NQ; ++j) acc[j][k] = mfma32<DT>(vt.v, pf[j], acc[j][k]);
      }
      wave_lds();

      if (__builtin_expect(odd, 0)) {
        const float nan = __uint_as_float(0x7fc00000u);
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
          for (int b = 0; b < B; ++b) {
            // lanes whose quarter begins in block b, or reaches it
            bool bad = nan_scale[u][0] == 255u && B * quarter / 4 == b;
            if constexpr (Tile::S == 2)
              bad |= nan_scale[u][1] == 255u && (B * quarter + B - 1) / 4 == b;
            uint64_t rows_nan = __ballot(bad && now[u]);
            rows_nan |= rows_nan >> 32;
            rows_nan |= rows_nan >> 16;
            uint32_t left = (uint32_t)rows_nan & 0xffffu;
            while (left) {
              const int tok = t0 + 16 * u + __builtin_ctz(left);
              left &= left - 1;
#pragma unroll
              for (int j = 0; j < NQ; ++j)
                if (tok < lim[j]) {
                  acc[j][2 * b] = f32x4{nan, nan, nan, nan};
                  acc[j][2 * b + 1] = f32x4{nan, nan, nan, nan};
                }
            }
          }
        }
      }
    };

    load_step();
    while (at < last) run_step();

    if (share == 1) {  // every wave has heads of its own: straight from the registers
#pragma unroll
      for (int j = 0; j < NQ; ++j) {
        l[j] += __shfl_xor(l[j], 16);
        l[j] += __shfl_xor(l[j], 32);
        const int64_t row = row0 + 16 * j + n;
        if (row >= rows) continue;
        const int64_t o = out_row(row, h);
        AttendScale sc{};
        if (g.splits == 1) {
          sc = attend_scale(a, o, m[j], l[j]);
          if (quarter == 0) a.lse[o] = sc.lse;
        } else if (quarter == 0) {
          g.part_ml[o * g.splits + split] = float2{m[j], l[j]};
        }
#pragma unroll
        for (int k = 0; k < NT; ++k) {
          const int d = 16 * k + 4 * quarter;
          if (g.splits == 1) attend_store<DT>(a, o, d, acc[j][k], sc);
          else *reinterpret_cast<f32x4*>(g.part_o + (o * g.splits + split) * D + d) = acc[j][k];
        }
      }
      continue;
    }
    // the waves of a head joined, 16 rows at a time
#pragma unroll
    for (int j = 0; j < NQ; ++j) {
      l[j] += __shfl_xor(l[j], 16);
      l[j] += __shfl_xor(l[j], 32);
      __syncthreads();
      if (quarter == 0) lds_ml[wave][n] = float2{m[j], l[j]};
      float* o = reinterpret_cast<float*>(lds) + wave * (D * 16);
#pragma unroll
      for (int k = 0; k < NT; ++k)
        *reinterpret_cast<f32x4*>(o + n * D + ((16 * k + 4 * quarter) ^ ((n & 7) << 2))) = acc[j][k];
      __syncthreads();
      const int col = (int)threadIdx.x >> 4;
      const int64_t row = row0 + 16 * j + col;
      if (row < rows) {
        for (int hh = 0; hh < g.wave_heads; ++hh) {
          float mt = ninf, lt = 0.0f, f[kAttendWaves];
#pragma unroll
          for (int w = 0; w < kAttendWaves; ++w)
            if (w % g.wave_heads == hh) mt = __builtin_fmaxf(mt, lds_ml[w][col].x);
#pragma unroll
          for (int w = 0; w < kAttendWaves; ++w) {
            const float2 ml = lds_ml[w][col];
            f[w] = w % g.wave_heads != hh || ml.y == 0.0f ? 0.0f : exp2_(ml.x - mt);
            if (w % g.wave_heads == hh) lt += ml.y * f[w];
          }
          const int64_t o = out_row(row, (int)blockIdx.y * g.wave_heads + hh);
          AttendScale sc{};
          if (g.splits == 1) {
            sc = attend_scale(a, o, mt, lt);
            if ((threadIdx.x & 15) == 0) a.lse[o] = sc.lse;
          } else if ((threadIdx.x & 15) == 0) {
            g.part_ml[o * g.splits + split] = float2{mt, lt};
          }
          for (int d = ((int)threadIdx.x & 15) * 4; d < D; d += 64) {
            f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int w = 0; w < kAttendWaves; ++w)
              if (w % g.wave_heads == hh)
                sum += *reinterpret_cast<const f32x4*>(reinterpret_cast<const float*>(lds) +
                                                       w * (D * 16) + col * D +
                                                       (d ^ ((col & 7) << 2))) * f[w];
            if (g.splits == 1) attend_store<DT>(a, o, d, sum, sc);
            else *reinterpret_cast<f32x4*>(g.part_o + (o * g.splits + split) * D + d) = sum;
          }
        }
      }
    }
    __syncthreads();
  }
}

// The splits of a row joined, in their order: a wave to a row, lane s weighing split s,
// then each lane summing columns.
template <int DT, int D>
__global__ __launch_bounds__(kThreads) void kv_mx_attend_join_kernel(AttendArgs g) {
  const dsr_attend_args& a = g.a;
  const AttendRequest rq = attend_request(a, (int)blockIdx.z);
  const int lane = (int)threadIdx.x % kWave;
  const int hq = __builtin_amdgcn_readfirstlane((int)(blockIdx.y * (kThreads / kWave) +
                                                      threadIdx.x / kWave));
  if (hq >= a.q_heads) return;
  const float ninf = -__builtin_inff();
  for (int i = rq.q0 + (int)blockIdx.x; i < rq.q1; i += (int)gridDim.x) {
    const int64_t at = (int64_t)i * a.q_heads + hq;
    int64_t seen = rq.tokens;
    if (a.limits && a.limits[i] < seen) seen = a.limits[i];
    int n = seen <= 0 ? 0 : (int)((seen + g.chunk - 1) / g.chunk);
    if (n > g.splits) n = g.splits;
    const float2* ml = g.part_ml + at * g.splits;
    const float* po = g.part_o + at * g.splits * D;
    // lane s weighs split s; kSum lanes to a row of columns, the others' rows are further
    // splits. The sums' loads go out before the weights are known.
    constexpr int kSum = D <= 64 ? 16 : D <= 128 ? 32 : 64, kRows = kWave / kSum, kFar = 8;
    const int sub = lane / kSum, col = lane % kSum * 4;
    const bool has = col < D;
    f32x4 o[kFar];
    auto fetch = [&](int s0) {
#pragma unroll
      for (int k = 0; k < kFar; ++k) {
        if (s0 + k * kRows >= n) break;
        const int s = s0 + k * kRows + sub;
        o[k] = *reinterpret_cast<const f32x4*>(po + (int64_t)(s < n ? s : 0) * D + (has ? col : 0));
      }
    };
    float m = ninf, l = 0.0f;
    f32x4 sum = {0.0f, 0.0f, 0.0f, 0.0f};
    if (n > 0) fetch(0);
    for (int s = lane; s < n; s += kWave) m = __builtin_fmaxf(m, ml[s].x);
#pragma unroll
    for (int k = 1; k < kWave; k <<= 1) m = __builtin_fmaxf(m, __shfl_xor(m, k));
    for (int s0 = 0; s0 < n; s0 += kWave) {
      float w = 0.0f;
      if (s0 + lane < n) {
        const float2 x = ml[s0 + lane];
        if (x.y != 0.0f) {  // NaN too
          w = exp2_(x.x - m);
          l += x.y * w;
        }
      }
      for (int s = s0; s < s0 + kWave && s < n; s += kFar * kRows) {
#pragma unroll
        for (int k = 0; k < kFar; ++k) {
          if (s + k * kRows >= n) break;
          const int at_s = s + k * kRows + sub;
          const float ws = __shfl(w, (at_s - s0) & (kWave - 1));
          if (at_s < n) sum += o[k] * ws;
        }
        if (s + kFar * kRows < n) fetch(s + kFar * kRows);
      }
    }
#pragma unroll
    for (int k = 1; k < kWave; k <<= 1) l += __shfl_xor(l, k);
#pragma unroll
    for (int k = kSum; k < kWave; k <<= 1)
#pragma unroll
      for (int e = 0; e < 4; ++e) sum[e] += __shfl_xor(sum[e], k);
    const AttendScale sc = attend_scale(a, at, m, l);
    if (lane == 0) a.lse[at] = sc.lse;
    if (lane < kSum && has) attend_store<DT>(a, at, col, sum, sc);
  }
}

}  // namespace
