// tb_wait.cuh — bounded device-side waits and the status word they report to.
// Each translation unit has its own status word; tb_device_status() reads and
// clears all of them.
#pragma once

#include <stdint.h>

#include "../../include/tb_gemm.h"
#include "tb_sm100.cuh"

static __device__ uint32_t g_tb_status = 0;

namespace {

constexpr long long kWaitBudgetCycles = 2000000000LL;  // ≈1 s at 1.9 GHz

constexpr uint32_t kSiteProducer = 1, kSiteMma = 2, kSiteEpilogue = 3, kSiteDrain = 4,
                   kSiteSelfTest = 5, kSiteFixer = 6, kSiteCluster = 7, kSiteScheduler = 8;

__device__ __forceinline__ void record_error(uint32_t code, uint32_t site) {
  const uint32_t v = (code << 24) | (site << 16) | (blockIdx.x & 0xFFFFu);
  atomicCAS(&g_tb_status, 0u, v);
}

// Bounded wait: false when the abort flag is up or the budget ran out.
__device__ __forceinline__ bool wait_bounded(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t site,
                                             long long budget = kWaitBudgetCycles) {
  if (tb::sm100::mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (true) {
    if (tb::sm100::mbar_try_wait(bar, parity)) return true;
    if (*abort_flag) return false;
    if (clock64() - t0 > budget) {
      record_error(TB_ERR_DEVICE_TIMEOUT, site);
      *abort_flag = 1;
      return false;
    }
  }
}

// Lane 0 waits (bounded), the result is broadcast so the warp stays converged.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t site,
                                          int lane, long long budget = kWaitBudgetCycles) {
  // Every lane probes first with the non-blocking test_wait: in the common
  // case (phase already complete) that is one probe, while a blocking
  // try_wait costs hundreds of cycles even on a completed phase (measured:
  // 142 → 118 cycles per MMA for a 128×128 tile, 154 → 132 for 128×256).
  // The warp goes by one answer: lanes that saw different ones would part here
  // and wait for each other at two instructions.
  if (__all_sync(0xffffffffu, tb::sm100::mbar_test_wait(bar, parity))) return true;
  int ok = 0;
  if (lane == 0) ok = wait_bounded(bar, parity, abort_flag, site, budget);
  return __shfl_sync(0xffffffffu, ok, 0) != 0;
}

// warp_wait without the blocking probe: the warp polls until the phase is
// complete, for waits whose every cycle is on the critical path (a blocked
// try_wait wakes up hundreds of cycles after the phase completes). CLUSTER:
// the barrier is arrived on by, or hands over data from, other CTAs of the cluster.
template <bool CLUSTER = false>
__device__ __forceinline__ bool warp_poll(uint32_t bar, uint32_t parity, volatile int* abort_flag, uint32_t site,
                                          int lane, long long budget = kWaitBudgetCycles) {
  auto probe = [&]() {
    if constexpr (CLUSTER) return tb::sm100::mbar_test_wait_cluster(bar, parity);
    else return tb::sm100::mbar_test_wait(bar, parity);
  };
  if (__all_sync(0xffffffffu, probe())) return true;
  const long long t0 = clock64();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (__all_sync(0xffffffffu, probe())) return true;
    int stop = 0;
    if (lane == 0) {
      stop = *abort_flag;
      if (!stop && clock64() - t0 > budget) {
        record_error(TB_ERR_DEVICE_TIMEOUT, site);
        *abort_flag = stop = 1;
      }
    }
    if (__shfl_sync(0xffffffffu, stop, 0)) return false;
  }
}

}  // namespace
