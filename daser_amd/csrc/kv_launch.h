// kv_launch.h -- launch helpers shared by the translation units of the kernels.

#pragma once

#include "kv_flat.h"

namespace {

inline bool aligned16(int64_t v) { return (v & 15) == 0; }
inline bool aligned16p(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

// Largest workgroup count of one launch: HIP caps gridDim.x * blockDim.x at
// 2^32 - 1 threads (16.7 M workgroups of 256). The DSR_TUNE_MAX_WG_PER_LAUNCH
// override lowers it, so that tests can exercise the split.
inline int64_t max_wg_per_launch() {
  int64_t m = 0xffffffffLL / kThreads / kXcds * kXcds;
  if (const int64_t t = tune(DSR_TUNE_MAX_WG_PER_LAUNCH)) {
    const int64_t v = t / kXcds * kXcds;
    if (v >= 2 * kXcds && v < m) m = v;
  }
  return m;
}

// Launches of a flat kernel over every piece of n_units units (one launch
// unless the workgroups exceed max_wg_per_launch()), `minor` the inner extent
// of the unit order: launch(map, grid). `chunk`: consecutive workgroups that stay
// on one XCD (0: dealt one by one; kEighths).
template <class F>
int launch_flat(int64_t n_units, int64_t pieces_per_unit, int64_t minor, uint32_t chunk, F launch) {
  constexpr int kWaves = kThreads / kWave;
  const int64_t total = n_units * pieces_per_unit;
  const int64_t per = max_wg_per_launch() * kWaves;
  for (int64_t g0 = 0; g0 < total; g0 += per) {
    const int64_t n = total - g0 < per ? total - g0 : per;
    unsigned grid = (unsigned)((n + kWaves - 1) / kWaves);
    FlatMap m;
    m.per_unit = fast_div((uint32_t)pieces_per_unit);
    m.minor = fast_div((uint32_t)minor);
    m.unit0 = (uint32_t)(g0 / pieces_per_unit);
    m.wave0 = (uint32_t)(g0 % pieces_per_unit);
    m.n_waves = (uint32_t)n;
    if (chunk == kEighths) grid = (grid + kXcds - 1) / kXcds * kXcds;  // the rest leave at once
    m.chunked = chunk == kEighths ? kEighthsBit | grid / kXcds
                : chunk == kChunk ? grid / (kXcds * kChunk) * (kXcds * kChunk) : 0;
    launch(m, grid);
    const int rc = (int)hipGetLastError();
    if (rc != 0) return rc;
  }
  return DSR_OK;
}

// Dynamic LDS that limits a kernel with `static_lds` bytes of static LDS to
// wg_per_cu workgroups per CU on the current device (0 if the capacity cannot
// be read). The capacity is read once per device.
constexpr int64_t kLdsGranule = 512;
constexpr int kMaxDevices = 64;
std::atomic<int> g_lds_per_cu[kMaxDevices];
inline size_t occupancy_lds(int wg_per_cu, int64_t static_lds) {
  int dev = 0;
  if (hipGetDevice(&dev) != hipSuccess || wg_per_cu <= 0) return 0;
  int lds = dev < kMaxDevices ? g_lds_per_cu[dev].load(std::memory_order_relaxed) : 0;
  if (lds <= 0) {
    if (hipDeviceGetAttribute(&lds, hipDeviceAttributeMaxSharedMemoryPerMultiprocessor,
                              dev) != hipSuccess || lds <= 0)
      return 0;
    if (dev < kMaxDevices) g_lds_per_cu[dev].store(lds, std::memory_order_relaxed);
  }
  // a workgroup's LDS (static plus dynamic) is allocated in 512-byte
  // granules: round its share down so that wg_per_cu of them fit
  const int64_t share = (int64_t)lds / wg_per_cu / kLdsGranule * kLdsGranule;
  const int64_t want = share - static_lds;
  return want > 0 ? (size_t)want : 0;
}

}  // namespace
