// Helpers of the C ABI translation units: workspace carving, dtype checks, stage timing.
#pragma once
#include <stdint.h>

#include <algorithm>

#include "host_util.h"
#include "stage_timer.h"

// Launch `expr` as pipeline stage `stage` (timed when the stage timer is on).
#define SB_STAGE(stage, expr)           \
  do {                                  \
    ::sb::StageScope _scope(stage, st); \
    SB_TRY(expr);                       \
  } while (0)

namespace sb {

// Bump allocator over the caller's workspace; with base == nullptr it only
// measures (the *_workspace_bytes queries run the same carve).
struct Carver {
  uint8_t* base;
  size_t off = 0;
  explicit Carver(void* b) : base(static_cast<uint8_t*>(b)) {}
  template <typename T>
  T* take(size_t n) {
    off = (off + 255) & ~size_t(255);
    T* p = base ? reinterpret_cast<T*>(base + off) : nullptr;
    off += n * sizeof(T);
    return p;
  }
  void* take_bytes(size_t n) { return take<uint8_t>(n); }
};

inline size_t esize(int dtype) {
  switch (dtype) {
    case STAGEML_F32:
    case STAGEML_I32:
      return 4;
    case STAGEML_BF16:
    case STAGEML_F16:
      return 2;
    case STAGEML_E4M3:
      return 1;
    case STAGEML_I64:
      return 8;
    default:
      return 0;
  }
}

inline bool is16(int dtype) { return dtype == STAGEML_BF16 || dtype == STAGEML_F16; }
inline bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

inline void carve_plan(Carver& c, int64_t P, int n_groups, stageml_moe_plan* plan) {
  const int64_t rows_cap = stageml_plan_rows_cap(P, n_groups);
  plan->rows_cap = rows_cap;
  plan->row_token = c.take<int32_t>(rows_cap);
  plan->row_tenant = c.take<int32_t>(rows_cap);
  plan->row_weight = c.take<float>(rows_cap);
  plan->row_pair = c.take<int32_t>(rows_cap);
  plan->pair_row = c.take<int32_t>(std::max<int64_t>(P, 1));
  plan->tile_group = c.take<int32_t>(rows_cap / 128);
  plan->group_offsets = c.take<int32_t>(n_groups + 1);
  plan->group_counts = c.take<int32_t>(n_groups);
  plan->num_tiles = c.take<int32_t>(1);
}

}  // namespace sb
