// The loop of a device-side wait that is bounded in time, apart from the instructions it polls and reads the clock with: it
// compiles for the host too, where a test gives it a barrier and a clock of its own.
#pragma once

#include <cstdint>

#if defined(__CUDACC__)
#define Q3X_WAIT_FUNCTION __device__ __forceinline__
#else
#define Q3X_WAIT_FUNCTION inline
#endif

namespace q3x {

constexpr uint64_t kMostPerPoll = 1000000;  // nanoseconds

// Polls until poll() holds (true), or until `limit` nanoseconds or `most_polls` polls have passed (false).  The clock is the
// wall's: it runs on while the process is switched off the GPU, between a poll that failed and the reading of the clock as
// well, and what is waited for stands still meanwhile.  So the time from one poll to the next counts for a millisecond at
// most: time away counts as one poll, and a barrier that was complete, or completes soon after, is seen by those that
// follow.  (A poll may hold its thread for some microseconds; were it longer than a millisecond, the bound would be as many
// polls as `limit` has milliseconds.)
template <class Poll, class Clock>
Q3X_WAIT_FUNCTION bool wait_in_time(const Poll& poll, const Clock& clock, uint64_t limit, uint32_t most_polls) {
  uint64_t last = clock(), waited = 0;
  for (uint32_t n = 0; n < most_polls; ++n) {
    if (poll()) return true;
    const uint64_t now = clock(), passed = now - last;
    waited += passed < kMostPerPoll ? passed : kMostPerPoll;
    if (waited > limit) return false;
    last = now;
  }
  return false;
}

}  // namespace q3x
