// kv_mx.hip -- launch policy and C ABI of the quantised records (kv_mx.h) and of the
// attention over them (kv_attend.h).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_attend.h"
#include "kv_launch.h"

namespace {

int64_t pad16(int64_t n) { return (n + 15) / 16 * 16; }

// Section bytes of one half; false for geometries that the format does not take.
bool mx_sections(int format, int block, int heads, int dim, int64_t* codes, int64_t* scales) {
  if (block <= 0 || heads <= 0 || dim <= 0 || dim % 32) return false;
  const __int128 elems = (__int128)block * heads * dim;
  if (elems * 2 > 0x7fffffffLL) return false;  // one buffer descriptor per cache page
  *codes = pad16((int64_t)elems / (format == DSR_MX_FP4 ? 2 : 1));
  *scales = pad16((int64_t)elems / 32);
  return true;
}

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

struct GatherPages {
  const MxArgs& a;
  const int32_t* ids;
  const int64_t* offs;
  const FlatMap& m;
  unsigned grid;
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
    kv_mx_gather_kernel<FMT, DT, HND><<<grid, kThreads, 0, s>>>(a, ids, offs, m);
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
  hipStream_t s;
  template <int FMT, int DT, bool HND>
  void operator()() const {
    if (style == DSR_ROPE_NEOX)
      kv_mx_scatter_kernel<FMT, DT, HND, DSR_ROPE_NEOX><<<grid, kThreads, 0, s>>>(a, r, ids, offs, m);
    else
      kv_mx_scatter_kernel<FMT, DT, HND, DSR_ROPE_GPTJ><<<grid, kThreads, 0, s>>>(a, r, ids, offs, m);
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

// ---------------------------------------------------------------------------
// Attention

constexpr int kMaxGridZ = 65535;

constexpr int kAttendWgs = 1024;      // workgroups that fill the chip
constexpr int kAttendMinChunk = 128;  // tokens: a step of each wave

// 16-row column tiles per workgroup.
int attend_nq(const AttendArgs& g) {
  const int64_t rows = (int64_t)(g.a.max_queries < 1 ? 1 : g.a.max_queries) * g.group;
  return rows <= 16 ? 1 : g.a.head_dim == 256 ? 2 : 4;
}

// The call's geometry checked and its launch planned; *work: there is something to do.
int attend_args(const dsr_attend_args* args, AttendArgs* g, bool* work) {
  *work = false;
  if (!args) return DSR_ERR_ARG;
  const dsr_attend_args& a = *args;
  if (a.n_req < 0 || a.n_q < 0 || a.n_pages < 0 || a.max_queries < 0 || a.max_context < 0 ||
      a.layer < 0 || a.staging_bytes < 0 || a.n_tables < 0 || a.workspace_bytes < 0)
    return DSR_ERR_ARG;
  if (a.format != DSR_MX_INT8 && a.format != DSR_MX_FP4) return DSR_ERR_ARG;
  if (a.dtype != DSR_DTYPE_BF16 && a.dtype != DSR_DTYPE_FP16) return DSR_ERR_ARG;
  int64_t codes, scales;
  if (!mx_sections(a.format, a.block_size, a.kv_heads, a.head_dim, &codes, &scales) ||
      2 * (codes + scales) > 0x7fffffffLL || a.layer_bytes < 2 * (codes + scales) ||
      a.block_size % 16 || a.q_heads <= 0 || a.q_heads % a.kv_heads || a.q_heads > 65535)
    return DSR_ERR_SHAPE;
  const int d = a.head_dim;
  if (d != 32 && d != 64 && d != 96 && d != 128 && d != 256) return DSR_ERR_SHAPE;
  if (a.rope_idx) {
    if (a.style != DSR_ROPE_NEOX && a.style != DSR_ROPE_GPTJ) return DSR_ERR_ARG;
    if (a.n_tables > 0 && !a.cos_sin) return DSR_ERR_ARG;
    if (a.rot_dim <= 0 || a.rot_dim > d || a.rot_dim % (a.style == DSR_ROPE_NEOX ? 16 : 8))
      return DSR_ERR_SHAPE;
  }
  if (a.n_req == 0 || a.n_q == 0) return DSR_OK;
  *work = true;
  *g = AttendArgs{};
  g->a = a;
  g->codes = (int)codes;
  g->scales = (int)scales;
  g->need = 2 * (codes + scales);
  g->group = a.q_heads / a.kv_heads;
  g->scale2 = a.scale * 1.4426950408889634f;
  // Tiles of query rows, and splits of the longest request's tokens where the tiles alone
  // do not fill the chip.
  const int64_t rows = (int64_t)(a.max_queries < 1 ? 1 : a.max_queries) * g->group;
  const int nq = attend_nq(*g);
  int64_t tiles = (rows + 16 * nq - 1) / (16 * nq);
  const int64_t nz = a.n_req < kMaxGridZ ? a.n_req : kMaxGridZ;
  const int64_t ctx = a.max_context < 1 ? 1 : a.max_context;
  int64_t splits = (kAttendWgs + tiles * a.kv_heads * nz - 1) / (tiles * a.kv_heads * nz);
  const int64_t most = (ctx + kAttendMinChunk - 1) / kAttendMinChunk;
  if (splits > most) splits = most;
  const int64_t chunk = ((ctx + splits - 1) / splits + kAttendMinChunk - 1) / kAttendMinChunk *
                        kAttendMinChunk;
  g->chunk = (int)(chunk < 0x40000000 ? chunk : 0x40000000);
  g->splits = (int)((ctx + g->chunk - 1) / g->chunk);
  // requests larger than the hints loop
  const int64_t room = max_wg_per_launch() / (a.kv_heads * nz * g->splits);
  g->tiles = (int)(tiles < 1 ? 1 : tiles > room ? (room < 1 ? 1 : room) : tiles);
  return DSR_OK;
}

int64_t attend_ml_bytes(const AttendArgs& g) {
  return pad16((int64_t)g.a.n_q * g.a.q_heads * g.splits * 8);
}
int64_t attend_bytes(const AttendArgs& g) {
  if (g.splits <= 1) return 0;
  return attend_ml_bytes(g) + (int64_t)g.a.n_q * g.a.q_heads * g.splits * g.a.head_dim * 4;
}

template <int FMT, int DT, int D, int NQ>
void launch_attend_as(const AttendArgs& g, dim3 grid, hipStream_t s) {
  if (g.a.rope_idx) kv_mx_attend_kernel<FMT, DT, D, NQ, true><<<grid, kThreads, 0, s>>>(g);
  else kv_mx_attend_kernel<FMT, DT, D, NQ, false><<<grid, kThreads, 0, s>>>(g);
}
template <int FMT, int DT>
void launch_attend_dims(const AttendArgs& g, dim3 grid, hipStream_t s) {
  const bool wide = attend_nq(g) > 1;
  switch (g.a.head_dim) {
#define DSR_ATTEND(D, N)                                          \
  case D:                                                         \
    if (wide) launch_attend_as<FMT, DT, D, N>(g, grid, s);        \
    else launch_attend_as<FMT, DT, D, 1>(g, grid, s);             \
    break;
    DSR_ATTEND(32, 4)
    DSR_ATTEND(64, 4)
    DSR_ATTEND(96, 4)
    DSR_ATTEND(128, 4)
    default:
      if (wide) launch_attend_as<FMT, DT, 256, 2>(g, grid, s);
      else launch_attend_as<FMT, DT, 256, 1>(g, grid, s);
#undef DSR_ATTEND
  }
}
void launch_attend(const AttendArgs& g, int n_req, hipStream_t s) {
  const dim3 grid((unsigned)(g.tiles * g.splits), (unsigned)g.a.kv_heads, (unsigned)n_req);
  const bool bf16 = g.a.dtype == DSR_DTYPE_BF16;
  if (g.a.format == DSR_MX_FP4) {
    if (bf16) launch_attend_dims<DSR_MX_FP4, DSR_DTYPE_BF16>(g, grid, s);
    else launch_attend_dims<DSR_MX_FP4, DSR_DTYPE_FP16>(g, grid, s);
  } else {
    if (bf16) launch_attend_dims<DSR_MX_INT8, DSR_DTYPE_BF16>(g, grid, s);
    else launch_attend_dims<DSR_MX_INT8, DSR_DTYPE_FP16>(g, grid, s);
  }
}
void launch_attend_join(const AttendArgs& g, int n_req, hipStream_t s) {
  const int per = kThreads / 16;
  const int64_t y = (g.a.q_heads + per - 1) / per;
  const int64_t room = max_wg_per_launch() / (y * n_req);
  int64_t x = g.a.max_queries < 1 ? 1 : g.a.max_queries;
  if (x > room) x = room < 1 ? 1 : room;
  const dim3 grid((unsigned)x, (unsigned)y, (unsigned)n_req);
  if (g.a.dtype == DSR_DTYPE_BF16)
    kv_mx_attend_join_kernel<DSR_DTYPE_BF16><<<grid, kThreads, 0, s>>>(g);
  else
    kv_mx_attend_join_kernel<DSR_DTYPE_FP16><<<grid, kThreads, 0, s>>>(g);
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
  return launch_flat((int64_t)n_pages * count, (a.vecs + kWave - 1) / kWave, count, 0,
                     [&](const FlatMap& m, unsigned grid) {
    mx_dispatch(args, GatherPages{a, page_ids, slot_offsets, m, grid, (hipStream_t)stream});
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
  return launch_flat((int64_t)n_pages * count, (a.vecs + kWave - 1) / kWave, n_pages, 0,
                     [&](const FlatMap& m, unsigned grid) {
    mx_dispatch(args, ScatterPages{a, r, rope ? rope->style : DSR_ROPE_NEOX, page_ids,
                                   slot_offsets, m, grid, (hipStream_t)stream});
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

int64_t dsr_attend_workspace(const dsr_attend_args* args) {
  AttendArgs g;
  bool work;
  const int rc = attend_args(args, &g, &work);
  return rc != DSR_OK ? rc : !work ? 0 : attend_bytes(g);
}

int dsr_attend_mx(const dsr_attend_args* args, dsr_stream_t stream) {
  AttendArgs g;
  bool work;
  const int rc = attend_args(args, &g, &work);
  if (rc != DSR_OK || !work) return rc;
  const dsr_attend_args& a = g.a;
  if (!a.q || !a.out || !a.lse || !a.q_start || !a.page_start || !a.context ||
      (a.n_pages > 0 && (!a.slot_offsets || !a.staging)) || !a.prior_out != !a.prior_lse)
    return DSR_ERR_ARG;
  if (!aligned16(a.q_row_stride) || !aligned16(a.q_head_stride) || !aligned16p(a.q) ||
      !aligned16p(a.out) || !aligned16p(a.prior_out) || !aligned16p(a.staging) ||
      !aligned16(a.layer_bytes) || !aligned16p(a.workspace))
    return DSR_ERR_ALIGN;
  const int64_t need = attend_bytes(g);
  if (need > a.workspace_bytes || (need > 0 && !a.workspace)) return DSR_ERR_ARG;
  g.part_ml = static_cast<float2*>(a.workspace);
  g.part_o = reinterpret_cast<float*>(static_cast<uint8_t*>(a.workspace) + attend_ml_bytes(g));
  hipStream_t s = (hipStream_t)stream;
  for (int r0 = 0; r0 < a.n_req; r0 += kMaxGridZ) {
    AttendArgs b = g;
    b.a.q_start += r0;
    b.a.page_start += r0;
    b.a.context += r0;
    const int n = a.n_req - r0 < kMaxGridZ ? a.n_req - r0 : kMaxGridZ;
    launch_attend(b, n, s);
    int e = (int)hipGetLastError();
    if (e != 0) return e;
    if (g.splits > 1) {
      launch_attend_join(b, n, s);
      if ((e = (int)hipGetLastError()) != 0) return e;
    }
  }
  return DSR_OK;
}

}  // extern "C"
