// What the selection kernels (select.hip) and the adjusted selection (adjust.hip)
// share: a candidate, and the advance of a decode batch by its selected ids.
#pragma once

#include "nd_internal.hpp"

namespace nd {
namespace sel {

constexpr uint32_t kNone = 0xFFFFFFFFu;

struct Best {
  float v;
  uint32_t order;  // position in candidate order; kNone = no candidate
};

}  // namespace sel
}  // namespace nd

// Feeds a row's selected id back as its next token, records it in the step
// history, appends it to the row's context and advances the row's position; the
// last row to finish (rows_done, zero between launches) advances the step
// counter.  One thread a row, once its workgroups have read the row's state.
__device__ __forceinline__ void nd_advance_row(const nd_select_advance& adv, uint32_t r,
                                               uint32_t batch, uint32_t id, double lp,
                                               uint32_t* rows_done) {
  const uint32_t step = __hip_atomic_load(adv.step, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  adv.tokens[r] = id;
  adv.positions[r] += 1;
  if (step < adv.history_steps) {
    adv.history[(size_t)step * batch + r] = id;
    adv.lp_history[(size_t)step * batch + r] = lp;
  }
  if (adv.context) {
    const uint32_t n = adv.context_lengths[r];
    if (n < adv.context_stride) {
      adv.context[(size_t)r * adv.context_stride + n] = id;
      adv.context_lengths[r] = n + 1;
    }
  }
  __builtin_amdgcn_s_waitcnt(0);  // this row's read of the step counter has completed
  if (__hip_atomic_fetch_add(rows_done, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) ==
      batch - 1) {
    __hip_atomic_store(rows_done, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    __hip_atomic_store(adv.step, step + 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
  }
}
