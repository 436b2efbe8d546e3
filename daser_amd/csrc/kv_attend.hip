// kv_attend.hip -- launch policy and C ABI of the attention over quantised records
// (kv_attend.h).

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "kv_attend.h"
#include "kv_launch.h"

namespace {

constexpr int kMaxGridZ = 65535;

// Workgroups that the splits aim at. One tile of rows: 2,048, some eight for each CU, so that
// ragged requests even out (decode batch of 64 x 8 heads: 1,536 150 us, 2,048 133, 3,072 142,
// 4,096 155). Several tiles: 512, which the chip holds at once (questions 512 79 us, 256 102,
// 1,024 96: each workgroup turns the queries and joins 32 rows).
constexpr int kAttendWgs = 2048, kAttendWideWgs = 512;
// Steps of heads and tokens from which a wave takes a head of its own: with as many waves as
// the chip holds, 16 tokens' worth of 64 steps each. Below, the waves of a workgroup share a
// head's tokens and join in LDS, which leaves the second kernel a quarter of the parts.
constexpr int64_t kAttendLarge = 256 * 16 * 64;
constexpr int kAttendMinChunk = 128;  // tokens of a split: a step of each wave

// Tiles of 16 rows per workgroup: what is dequantised serves them all, and their
// accumulators leave room for two waves a SIMD. 4 x 64 queries over 4,096 tokens, 2 -> 4 tiles:
// Llama-3-8B mxfp4 48 -> 72 us, mxint8 62 -> 81, Phi-3-mini 57 -> 73; head_dim 64: Llama-3.2-1B
// mxfp4 36.6 -> 37.3, Qwen2-0.5B mxint8 35.5 -> 28.3. Gemma-2-9B (256), 1 -> 2: 89 -> 73; its
// moved chunks, with both halves of the queries, do not fit twice.
int attend_nq(const AttendArgs& g) {
  const int64_t rows = (int64_t)(g.a.max_queries < 1 ? 1 : g.a.max_queries) * g.group;
  const int d = g.a.head_dim;
  if (rows <= 16 || (d == 256 && g.a.rope_idx)) return 1;
  return d >= 96 ? 2 : 4;
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
  if ((int64_t)a.n_q * a.q_heads > 0x7fffffffLL) return DSR_ERR_ARG;  // rows are 32-bit numbers
  *work = true;
  *g = AttendArgs{};
  g->a = a;
  g->codes = (int)codes;
  g->scales = (int)scales;
  g->need = 2 * (codes + scales);
  g->group = a.q_heads / a.kv_heads;
  g->scale2 = a.scale * 1.4426950408889634f;
  g->by_block = fast_div((uint32_t)a.block_size);
  // Tiles of query rows, and splits of the longest request's tokens where the tiles alone
  // do not fill the chip.
  const int64_t rows = (int64_t)(a.max_queries < 1 ? 1 : a.max_queries) * g->group;
  const int nq = attend_nq(*g);
  int64_t tiles = (rows + 16 * nq - 1) / (16 * nq);
  const int64_t nz = a.n_req < kMaxGridZ ? a.n_req : kMaxGridZ;
  const int64_t ctx = a.max_context < 1 ? 1 : a.max_context;
  g->wave_heads = 1;
  if (nq == 1 && nz * a.kv_heads * ctx >= kAttendLarge)
    g->wave_heads = a.kv_heads % 4 == 0 ? 4 : a.kv_heads % 2 == 0 ? 2 : 1;
  const int64_t least = kAttendMinChunk / g->wave_heads;
  const int64_t wgs = tiles * (a.kv_heads / g->wave_heads) * nz;
  int64_t splits = ((nq == 1 ? kAttendWgs : kAttendWideWgs) + wgs - 1) / wgs;
  const int64_t most = (ctx + least - 1) / least;
  if (splits > most) splits = most;
  const int64_t chunk = ((ctx + splits - 1) / splits + least - 1) / least * least;
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

template <int FMT, int DT, int D>
void launch_attend_as(const AttendArgs& g, dim3 grid, hipStream_t s) {
  constexpr int kWide = D >= 96 ? 2 : 4, kWideRope = D == 256 ? 1 : kWide;
  if (g.a.rope_idx) {
    if (attend_nq(g) > 1)
      kv_mx_attend_kernel<FMT, DT, D, kWideRope, true><<<grid, kThreads, 0, s>>>(g);
    else
      kv_mx_attend_kernel<FMT, DT, D, 1, true><<<grid, kThreads, 0, s>>>(g);
  } else {
    if (attend_nq(g) > 1)
      kv_mx_attend_kernel<FMT, DT, D, kWide, false><<<grid, kThreads, 0, s>>>(g);
    else
      kv_mx_attend_kernel<FMT, DT, D, 1, false><<<grid, kThreads, 0, s>>>(g);
  }
}
template <int FMT, int DT>
void launch_attend_dims(const AttendArgs& g, dim3 grid, hipStream_t s) {
  switch (g.a.head_dim) {
    case 32: launch_attend_as<FMT, DT, 32>(g, grid, s); break;
    case 64: launch_attend_as<FMT, DT, 64>(g, grid, s); break;
    case 96: launch_attend_as<FMT, DT, 96>(g, grid, s); break;
    case 128: launch_attend_as<FMT, DT, 128>(g, grid, s); break;
    default: launch_attend_as<FMT, DT, 256>(g, grid, s);
  }
}
void launch_attend(const AttendArgs& g, int n_req, hipStream_t s) {
  // An odd number of workgroups to a (request, heads): the XCDs are dealt workgroups in
  // turn, and with an even number the first splits, which every request has, fall to some
  // of them and the last, which few have, to others (decode batch 174 -> 137 us). Several
  // tiles of rows are cut to fill the chip once: one more would start a second round
  // (questions 72 -> 98 us).
  unsigned x = (unsigned)(g.tiles * g.splits);
  if (attend_nq(g) == 1) x |= 1u;
  const dim3 grid(x, (unsigned)(g.a.kv_heads / g.wave_heads), (unsigned)n_req);
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
  const int per = kThreads / kWave;
  const int64_t y = (g.a.q_heads + per - 1) / per;
  const int64_t room = max_wg_per_launch() / (y * n_req);
  int64_t x = g.a.max_queries < 1 ? 1 : g.a.max_queries;
  if (x > room) x = room < 1 ? 1 : room;
  const dim3 grid((unsigned)x, (unsigned)y, (unsigned)n_req);
  const bool bf16 = g.a.dtype == DSR_DTYPE_BF16;
#define DSR_JOIN(D)                                                                       \
  if (bf16) kv_mx_attend_join_kernel<DSR_DTYPE_BF16, D><<<grid, kThreads, 0, s>>>(g);      \
  else kv_mx_attend_join_kernel<DSR_DTYPE_FP16, D><<<grid, kThreads, 0, s>>>(g)
  switch (g.a.head_dim) {
    case 32: DSR_JOIN(32); break;
    case 64: DSR_JOIN(64); break;
    case 96: DSR_JOIN(96); break;
    case 128: DSR_JOIN(128); break;
    default: DSR_JOIN(256);
  }
#undef DSR_JOIN
}

}  // namespace

extern "C" {

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
      !aligned16(a.layer_bytes) || !aligned16p(a.workspace) || !aligned16p(a.cos_sin))
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
