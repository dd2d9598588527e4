// How a kernel that gave up a bounded wait says so.
#pragma once
#include "kernels.h"
#include "ptx.cuh"

namespace gonn {
namespace {

// Raises the CTA's abort flag; true for the one role that raised it.  Only that role reports:
// the roles that leave because they SAW the flag would otherwise overwrite the cause with
// their own, later, wait (the status words live in mapped host memory, where "write only if
// still zero" cannot tell a report of a microsecond ago from none).
__device__ __forceinline__ bool first_to_give_up(volatile uint32_t* abort_flag) {
  return atomicExch(const_cast<uint32_t*>(abort_flag), 1u) == 0u;
}

__device__ __forceinline__ void report(GemmStatus* st, uint32_t code, uint32_t where,
                                       uint32_t tile, uint32_t kb) {
  // `st` may be page-locked host memory mapped into the device: plain stores
  // only (the first reporter wins most of the time, which is all that is needed).
  volatile GemmStatus* v = st;
  if (v->code == 0u) {
    v->where = where;
    v->tile = tile;
    v->kblock = kb;
    v->code = code;
  }
}

// Before a block whose waits may have run out leaves.
__device__ __forceinline__ void wait_out(volatile uint32_t* abort_flag) {
  if (!*abort_flag) return;
  // a role gave up: give copies and MMAs in flight time to land
  const uint64_t t0 = ptx::globaltimer_ns();
  for (uint32_t i = 0; i < (1u << 16); ++i) {
    if (ptx::globaltimer_ns() - t0 > 2000000ull) break;
    __nanosleep(1000);
  }
}

}  // namespace
}  // namespace gonn
