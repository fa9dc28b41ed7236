// objb_launch.h -- host-side planning of the pipelined row-streaming kernels.
#pragma once

#include <cuda_runtime.h>

#include <cstddef>
#include <cstdint>
#include <utility>

namespace objb {

// Mirror of dev::RowLayout (same field order; the device struct is passed by
// value as a kernel argument).
struct RowLayoutHost {
  int rows, cols;
  int nblocks;
  int row_bytes;
  int srow_bytes;
  int nseg;
  int lpr;
  int rpw;
  int ngrp;
  int tstage;
  int nslots;
  int stage_bytes;
};

struct DeviceProps {
  int sm_count = 0;
  int max_smem_optin = 0;
  size_t l2_bytes = 0;
  int cc_major = 0, cc_minor = 0;
};

// Cached per-device properties (queried once per device).
int device_props(int device, DeviceProps* out);
int current_device(int* dev);

// Plans the row streaming of a rows x cols matrix whose packed rows are
// `row_bytes` (+ `srow_bytes` of split scales) long, with lane tiles covering
// `blocks_per_lane` blocks.  `dual` doubles the per-stage bytes (two matrices
// per stage).  Returns false when the shape cannot use the bulk-copy path.
// `smem_budget` bounds the stage ring: plain GEMVs (one matrix per call, calls
// back to back) keep the default; the MoE and FFN programs take the larger
// budget, where a third stage of wide rows shortens each expert's ramp.
constexpr int kGemvSmemBudget = 200 * 1024;
constexpr int kMoeSmemBudget = 226 * 1024;
bool plan_rows(int rows, int cols, int row_bytes, int srow_bytes, int blocks_per_lane, bool dual,
               int max_consumer_warps, RowLayoutHost* L, int smem_budget = kGemvSmemBudget);
// The same with the lanes a row spreads over given directly.
bool plan_rows_lanes(int rows, int cols, int row_bytes, int srow_bytes, int lanes, bool dual, int max_consumer_warps,
                     RowLayoutHost* L, int smem_budget = kGemvSmemBudget);

size_t pipe_smem_bytes(const RowLayoutHost& L);

// Opts a kernel into large dynamic shared memory once per (kernel, device).
int ensure_smem_attr_ptr(const void* kernel, int device, size_t bytes);

inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15u) == 0; }

// Rows of `width` bytes, `pitch` (>= width) apart; p null: nothing.
struct Rows {
  const void* p;
  size_t rows, width, pitch;
};
// Whether two arrays share a byte.  Rows of different pitches that lie among one
// another are not looked through: false.
inline bool overlap(Rows a, Rows b) {
  if (!a.p || !b.p || !a.rows || !b.rows || !a.width || !b.width) return false;
  for (Rows* r : {&a, &b})
    if (r->pitch == r->width) r->width *= r->rows, r->rows = 1;
  auto begin = [](const Rows& r) { return reinterpret_cast<uintptr_t>(r.p); };
  auto end = [&](const Rows& r) { return begin(r) + (r.rows - 1) * r.pitch + r.width; };
  if (begin(a) >= end(b) || begin(b) >= end(a)) return false;
  if (a.rows == 1) std::swap(a, b);
  if (a.rows == 1) return true;
  if (b.rows > 1 && b.pitch != a.pitch) return false;
  // b's first row from the start of a's row at or before it: within that row, or into the next
  const size_t pitch = a.pitch;
  const size_t d = begin(b) >= begin(a) ? (begin(b) - begin(a)) % pitch : (pitch - (begin(a) - begin(b)) % pitch) % pitch;
  return d < a.width || d + b.width > pitch;
}

}  // namespace objb
