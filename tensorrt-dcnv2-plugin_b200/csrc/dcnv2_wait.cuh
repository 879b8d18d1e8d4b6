// dcnv2_wait.cuh — the bounded mbarrier wait of every kernel of this library.
#pragma once
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/dcnv2.h"
#include "ptx_sm100.cuh"

namespace dcnv2 {

// ------------------------------------------------------------------ bounded mbarrier wait
// Waits for the phase of `bar` with the given parity. Gives up after timeout_ns (sets the CTA
// abort flag and the device error word) or as soon as another role of this CTA has aborted;
// both are checked every 16 tries so that a waiting warp issues few instructions.
// SLEEP_NS > 0 adds a nanosleep between tries; SLEEP_NS < 0 (kSuspend) lets the hardware suspend
// the thread until the phase completes; 0 spins (the MMA issuer, whose wake-up latency is on the
// critical path). Waiting warps that do not spin leave the issue slots to the working ones.
// CL selects a cluster-scope acquire (barriers that the peer CTA of a pair arrives on).
// Where the wait is for a role whose own work may take long, `moved` is a count that this role
// steps as it gets on: the time limit starts again, once, and then whenever the count has changed
// (it is read only when the limit is over, so that a wait that ends in time costs nothing more).
constexpr int kSuspend = -1;
struct WaitCtx {
  unsigned long long timeout_ns;
  int* err;                  // device error word
  volatile int* abort_flag;  // this CTA's abort flag (shared memory)
  volatile int* moved = nullptr;
};
template <int SLEEP_NS = 0, bool CL = false>
__device__ __forceinline__ bool wait_bar(uint32_t bar, uint32_t parity, const WaitCtx& w,
                                         int code) {
  if (CL ? ptx::mbar_try_wait_cluster(bar, parity) : ptx::mbar_try_wait(bar, parity)) return true;
  uint64_t t0 = ptx::global_timer_ns();
  int seen = -1;  // (counts are not negative)
  for (uint32_t n = 1;; ++n) {
    if constexpr (SLEEP_NS > 0) __nanosleep(static_cast<unsigned>(SLEEP_NS));
    if constexpr (CL) {
      if (ptx::mbar_try_wait_cluster(bar, parity)) return true;
    } else if constexpr (SLEEP_NS < 0) {
      if (ptx::mbar_try_wait_sleep(bar, parity, 1000000u)) return true;
    } else {
      if (ptx::mbar_try_wait(bar, parity)) return true;
    }
    if ((n & 15u) == 0) {
      if (*w.abort_flag) return false;
      if (ptx::global_timer_ns() - t0 > w.timeout_ns) {
        if (w.moved) {
          const int now = *w.moved;
          if (now != seen) {
            seen = now;
            t0 = ptx::global_timer_ns();
            continue;
          }
        }
        *w.abort_flag = 1;
        atomicOr(w.err, code);
        return false;
      }
    }
  }
}

// The same wait for what a kernel itself still has in flight (copies, MMAs) before it ends or frees
// tensor memory: neither an abort nor a shorter limit of the other waits cuts it short, only its
// own limit, which no copy or MMA that still runs comes near.
constexpr unsigned long long kDrainNs = 2000000000ull;
__device__ __forceinline__ bool drain_bar(uint32_t bar, uint32_t parity, const WaitCtx& w) {
  const uint64_t t0 = ptx::global_timer_ns();
  for (;;) {
    if (ptx::mbar_try_wait(bar, parity)) return true;
    if (ptx::global_timer_ns() - t0 > kDrainNs) {
      *w.abort_flag = 1;
      atomicOr(w.err, DCNV2_DEVERR_TIMEOUT_DRAIN);
      return false;
    }
  }
}

}  // namespace dcnv2
