// kv_mx.hip -- launch policy and C ABI of the quantised records (kv_mx.h).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_launch.h"
#include "kv_mx.h"

namespace {

// Checks a call's caches, records and layers; fills the kernels' arguments.
int mx_args(const dsr_mx_args* in, int first, int count, const void* t1, const void* t2, int n,
            MxArgs* a) {
  if (!in || n < 0 || first < 0 || count < 0 || in->n_layers < 0 || in->layer0 < 0 ||
      first > in->n_layers - count || in->num_blocks < 0 || in->staging_bytes < 0)
    return DSR_ERR_ARG;
  if (in->format != DSR_MX_INT8 && in->format != DSR_MX_FP4) return DSR_ERR_ARG;
  if (in->dtype != DSR_DTYPE_BF16 && in->dtype != DSR_DTYPE_FP16) return DSR_ERR_ARG;
  if (in->k_layout == DSR_K_KX) return DSR_ERR_SHAPE;
  if (in->k_layout != DSR_K_NHD && in->k_layout != DSR_K_HND) return DSR_ERR_ARG;
  int64_t codes, scales;
  if (!mx_sections(in->format, in->block_size, in->num_heads, in->head_dim, &codes, &scales) ||
      in->layer_bytes < 2 * (codes + scales))
    return DSR_ERR_SHAPE;
  if (n == 0 || count == 0) return DSR_OK;
  if (!in->layer_base || !in->staging || !t1 || !t2) return DSR_ERR_ARG;
  if (!aligned16(in->kv_stride) || !aligned16(in->page_stride) || !aligned16(in->layer_bytes) ||
      !aligned16p(in->staging))
    return DSR_ERR_ALIGN;
  *a = MxArgs{};
  a->layer_base = in->layer_base;
  a->kv_stride = in->kv_stride;
  a->page_stride = in->page_stride;
  a->num_blocks = in->num_blocks;
  a->staging = static_cast<uint8_t*>(in->staging);
  a->staging_bytes = in->staging_bytes;
  a->layer_bytes = in->layer_bytes;
  a->need = 2 * (codes + scales);
  a->page_bytes = 2LL * in->block_size * in->num_heads * in->head_dim;
  a->layer0 = in->layer0;
  a->first = first;
  a->vecs = (int)(a->page_bytes >> 4);
  a->codes = (int)codes;
  a->scales = (int)scales;
  a->heads = in->num_heads;
  a->block = in->block_size;
  a->block_shift = in->block_size & (in->block_size - 1) ? -1 : __builtin_ctz((unsigned)in->block_size);
  a->row_vecs = fast_div((uint32_t)in->head_dim / 8);
  a->by_block = fast_div((uint32_t)in->block_size);
  a->by_heads = fast_div((uint32_t)in->num_heads);
  return DSR_OK;
}

int mx_rope(const dsr_mx_args* in, const dsr_mx_rope* rope, MxRope* r) {
  *r = MxRope{};
  if (!rope) return DSR_OK;
  if (rope->style != DSR_ROPE_NEOX && rope->style != DSR_ROPE_GPTJ) return DSR_ERR_ARG;
  if (rope->n_tables < 0 || (rope->layer_group && rope->n_groups < 1)) return DSR_ERR_ARG;
  if (!rope->rope_idx || (rope->n_tables > 0 && !rope->cos_sin)) return DSR_ERR_ARG;
  if (!aligned16p(rope->cos_sin)) return DSR_ERR_ALIGN;
  const int rd = rope->rot_dim;
  if (rd <= 0 || rd > in->head_dim || rd % (rope->style == DSR_ROPE_NEOX ? 16 : 8))
    return DSR_ERR_SHAPE;
  r->cos_sin = reinterpret_cast<const float2*>(rope->cos_sin);
  r->rope_idx = rope->rope_idx;
  r->layer_group = rope->layer_group;
  r->n_tables = rope->n_tables;
  r->n_groups = rope->n_groups;
  r->rot_vecs = rd / 8;
  r->half_vecs = rope->style == DSR_ROPE_NEOX ? rd / 16 : 0;
  return DSR_OK;
}

// f<FMT, DT, HND>() of the call's format, type and layout.
template <class F>
void mx_dispatch(const dsr_mx_args* in, F f) {
#define DSR_MX_HND(FMT, DT)                                                \
  if (in->k_layout == DSR_K_HND) f.template operator()<FMT, DT, true>();   \
  else f.template operator()<FMT, DT, false>()
#define DSR_MX_DT(FMT)                                                 \
  if (in->dtype == DSR_DTYPE_BF16) { DSR_MX_HND(FMT, DSR_DTYPE_BF16); } \
  else { DSR_MX_HND(FMT, DSR_DTYPE_FP16); }
  if (in->format == DSR_MX_FP4) {
    DSR_MX_DT(DSR_MX_FP4)
  } else {
    DSR_MX_DT(DSR_MX_INT8)
  }
#undef DSR_MX_DT
#undef DSR_MX_HND
}

// Launch shape of the page form, by the bytes of cache it moves. Over 200 MiB (as the copies'
// copy_shape) the stores are nt sc0 sc1 in chunks of workgroups. Llama-3-8B, 79,906 tokens
// saved in mxint8 (15.9 GB) and loaded, Llama-3-8B 81,920 loaded rotated (16.3 GB), fp16
// Qwen2.5-7B head-major from mxfp4 (1.70 GB):
//   save: 4 pieces a wave, 4 workgroups a CU 2.72 ms (5.83 TB/s); 1 piece 3.77, 2 2.75, 8 2.89,
//     6 a CU 2.79; stores nt 2.77, sc0 sc1 2.95;
//   load: 6 a CU 2.68 ms (5.92 TB/s), 4 2.86, 5 2.86, 8 2.74; nt 2.72, sc0 sc1 2.93. From e2m1,
//     a quarter of whose bytes are reads, and where K turns, a wave's life is latency, not
//     bytes: 8 a CU 287 us (322 at 6, 366 at 4) and 3.14 ms (3.36 at 6, 4.06 at 4).
// Below, nt and one piece a wave: the launch is over with its first waves.
constexpr int64_t kMxLarge = 200 << 20;
constexpr int kMxPieces = 4, kMxGatherWgPerCu = 4, kMxScatterWgPerCu = 6, kMxTurnWgPerCu = 8,
              kMxPairsWgPerCu = 5;
struct MxShape {
  bool large;
  uint32_t chunk;
  int pieces;  // vectors of 64 per wave
};
MxShape mx_shape(const MxArgs& a, int64_t units) {
  const bool large = 2 * a.page_bytes * units > kMxLarge;
  return {large, large ? kChunk : 0u, large ? kMxPieces : 1};
}

struct GatherPages {
  const MxArgs& a;
  const int32_t* ids;
  const int64_t* offs;
  const FlatMap& m;
  unsigned grid;
  size_t dyn;
  bool large;
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
    if (large)
      kv_mx_gather_kernel<FMT, DT, HND, kMxPieces, kStoreNtSc><<<grid, kThreads, dyn, s>>>(a, ids, offs, m);
    else
      kv_mx_gather_kernel<FMT, DT, HND, 1, kStoreNt><<<grid, kThreads, dyn, s>>>(a, ids, offs, m);
  }
};
struct ScatterPages {
  const MxArgs& a;
  const MxRope& r;
  int style;
  const int32_t* ids;
  const int64_t* offs;
  const FlatMap& m;
  unsigned grid;
  size_t dyn;
  bool large;
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
#define DSR_MX_SCATTER(STYLE, POLICY) \
  kv_mx_scatter_kernel<FMT, DT, HND, STYLE, POLICY><<<grid, kThreads, dyn, s>>>(a, r, ids, offs, m)
    if (style == DSR_ROPE_NEOX) {
      if (large) DSR_MX_SCATTER(DSR_ROPE_NEOX, kStoreNtSc);
      else DSR_MX_SCATTER(DSR_ROPE_NEOX, kStoreNt);
    } else {
      if (large) DSR_MX_SCATTER(DSR_ROPE_GPTJ, kStoreNtSc);
      else DSR_MX_SCATTER(DSR_ROPE_GPTJ, kStoreNt);
    }
#undef DSR_MX_SCATTER
  }
};
struct ScatterPairs {
  const MxArgs& a;
  const MxRope& r;
  const int32_t* ids;
  const int64_t* offs;
  const FlatMap& m;
  unsigned grid;
  size_t dyn;
  bool large;
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
    const FastDiv half = fast_div((uint32_t)r.half_vecs);
    if (large)
      kv_mx_scatter_pairs_kernel<FMT, DT, HND, kStoreNtSc>
          <<<grid, kThreads, dyn, s>>>(a, r, ids, offs, m, half);
    else
      kv_mx_scatter_pairs_kernel<FMT, DT, HND, kStoreNt>
          <<<grid, kThreads, dyn, s>>>(a, r, ids, offs, m, half);
  }
};
struct Tokens {
  const MxArgs& a;
  const MxRope* r;  // null: gather
  int style;
  const int64_t* slots;
  const int64_t* rows;
  uint32_t n;
  FastDiv per;
  dim3 grid;
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
    if (!r)
      kv_mx_gather_slots_kernel<FMT, DT, HND><<<grid, kThreads, 0, s>>>(a, slots, rows, n, per);
    else if (style == DSR_ROPE_NEOX)
      kv_mx_scatter_slots_kernel<FMT, DT, HND, DSR_ROPE_NEOX>
          <<<grid, kThreads, 0, s>>>(a, *r, slots, rows, n, per);
    else
      kv_mx_scatter_slots_kernel<FMT, DT, HND, DSR_ROPE_GPTJ>
          <<<grid, kThreads, 0, s>>>(a, *r, slots, rows, n, per);
  }
};

// Token-form launches: tokens in ranges whose vectors, and layers in ranges that, one
// grid holds.
int launch_tokens(const dsr_mx_args* in, MxArgs a, const MxRope* rope, int style, int count,
                  const int64_t* slots, const int64_t* rows, int n, hipStream_t s) {
  const int64_t vecs = (int64_t)in->num_heads * in->head_dim / 8;  // of one token
  const int64_t wgs = max_wg_per_launch();
  const int layers = (int)(wgs < 65535 ? wgs : 65535);
  int64_t per = wgs / (count < layers ? count : layers) * kThreads / vecs;
  if (per < 1) per = 1;
  MxRope r = rope ? *rope : MxRope{};
  for (int l0 = 0; l0 < count; l0 += layers) {
    const int nl = count - l0 < layers ? count - l0 : layers;
    MxArgs b = a;
    b.first += l0;
    for (int64_t t0 = 0; t0 < n; t0 += per) {
      const int64_t nt = n - t0 < per ? n - t0 : per;
      const dim3 grid((unsigned)((nt * vecs + kThreads - 1) / kThreads), (unsigned)nl);
      if (rope) r.rope_idx = rope->rope_idx ? rope->rope_idx + t0 : nullptr;
      mx_dispatch(in, Tokens{b, rope ? &r : nullptr, style, slots + t0, rows + t0, (uint32_t)nt,
                             fast_div((uint32_t)vecs), grid, s});
      const int rc = (int)hipGetLastError();
      if (rc != 0) return rc;
    }
  }
  return DSR_OK;
}

}  // namespace

extern "C" {

int64_t dsr_mx_layer_bytes(int format, int block_size, int num_heads, int head_dim) {
  if (format != DSR_MX_INT8 && format != DSR_MX_FP4) return DSR_ERR_ARG;
  int64_t codes, scales;
  if (!mx_sections(format, block_size, num_heads, head_dim, &codes, &scales)) return DSR_ERR_SHAPE;
  return 2 * (codes + scales);
}

int dsr_gather_mx(const dsr_mx_args* args, int first, int count, const int32_t* page_ids,
                  const int64_t* slot_offsets, int n_pages, dsr_stream_t stream) {
  MxArgs a;
  const int rc = mx_args(args, first, count, page_ids, slot_offsets, n_pages, &a);
  if (rc != DSR_OK || n_pages == 0 || count == 0) return rc;
  if ((int64_t)n_pages * count > 0x7fffffffLL) return DSR_ERR_ARG;
  const MxShape c = mx_shape(a, (int64_t)n_pages * count);
  const int64_t per = kWave * c.pieces;
  const int cb = args->format == DSR_MX_FP4 ? 4 : 8;
  const size_t dyn = occupancy_lds(kMxGatherWgPerCu, (kThreads / kWave) * (per * cb + c.pieces * 16));
  return launch_flat((int64_t)n_pages * count, (a.vecs + per - 1) / per, count, c.chunk,
                     [&](const FlatMap& m, unsigned grid) {
    mx_dispatch(args, GatherPages{a, page_ids, slot_offsets, m, grid, dyn, c.large,
                                  (hipStream_t)stream});
  });
}

int dsr_scatter_mx(const dsr_mx_args* args, int first, int count, const int32_t* page_ids,
                   const int64_t* slot_offsets, int n_pages, const dsr_mx_rope* rope,
                   dsr_stream_t stream) {
  MxArgs a;
  MxRope r;
  int rc = mx_args(args, first, count, page_ids, slot_offsets, n_pages, &a);
  if (rc != DSR_OK || n_pages == 0 || count == 0) return rc;
  if ((rc = mx_rope(args, rope, &r)) != DSR_OK) return rc;
  if ((int64_t)n_pages * count > 0x7fffffffLL) return DSR_ERR_ARG;
  const MxShape c = mx_shape(a, (int64_t)n_pages * count);
  if (rope && rope->style == DSR_ROPE_NEOX && rope->rot_dim == args->head_dim) {
    const size_t lds = occupancy_lds(kMxPairsWgPerCu, 0);
    return launch_flat((int64_t)n_pages * count, (a.vecs / 2 + kWave - 1) / kWave, n_pages, c.chunk,
                       [&](const FlatMap& m, unsigned grid) {
      mx_dispatch(args, ScatterPairs{a, r, page_ids, slot_offsets, m, grid, lds, c.large,
                                     (hipStream_t)stream});
    });
  }
  const size_t dyn = occupancy_lds(rope || args->format == DSR_MX_FP4 ? kMxTurnWgPerCu : kMxScatterWgPerCu, 0);
  return launch_flat((int64_t)n_pages * count, (a.vecs + kWave - 1) / kWave, n_pages, c.chunk,
                     [&](const FlatMap& m, unsigned grid) {
    mx_dispatch(args, ScatterPages{a, r, rope ? rope->style : DSR_ROPE_NEOX, page_ids,
                                   slot_offsets, m, grid, dyn, c.large, (hipStream_t)stream});
  });
}

int dsr_gather_slots_mx(const dsr_mx_args* args, int first, int count,
                        const int64_t* slot_mapping, const int64_t* record_rows, int n_tokens,
                        dsr_stream_t stream) {
  MxArgs a;
  const int rc = mx_args(args, first, count, slot_mapping, record_rows, n_tokens, &a);
  if (rc != DSR_OK || n_tokens == 0 || count == 0) return rc;
  return launch_tokens(args, a, nullptr, 0, count, slot_mapping, record_rows, n_tokens,
                       (hipStream_t)stream);
}

int dsr_scatter_slots_mx(const dsr_mx_args* args, int first, int count,
                         const int64_t* slot_mapping, const int64_t* record_rows, int n_tokens,
                         const dsr_mx_rope* rope, dsr_stream_t stream) {
  MxArgs a;
  MxRope r;
  int rc = mx_args(args, first, count, slot_mapping, record_rows, n_tokens, &a);
  if (rc != DSR_OK || n_tokens == 0 || count == 0) return rc;
  if ((rc = mx_rope(args, rope, &r)) != DSR_OK) return rc;
  return launch_tokens(args, a, &r, rope ? rope->style : DSR_ROPE_NEOX, count, slot_mapping,
                       record_rows, n_tokens, (hipStream_t)stream);
}

}  // extern "C"
