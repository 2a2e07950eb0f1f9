// The loop of the bounded device-side waits (csrc/bounded_wait.hpp) with a barrier and a clock made up on the host.
#include <cstdint>
#include <cstdio>

#include "bounded_wait.hpp"

static int failures = 0;
#define EXPECT(cond)                                                  \
  do {                                                                \
    if (!(cond)) {                                                    \
      ++failures;                                                     \
      std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #cond);     \
    }                                                                 \
  } while (0)

namespace {

constexpr std::uint64_t kMs = 1000000, kLimit = 200 * kMs;
constexpr std::uint32_t kPolls = 1U << 20;

// Every reading of the clock is `step` after the last; the reading number `away_at` comes `away` later than that.
struct Clock {
  std::uint64_t step, away_at, away;
  mutable std::uint64_t now = 1000, readings = 0;
  std::uint64_t operator()() const {
    now += step + (readings == away_at ? away : 0);
    ++readings;
    return now;
  }
};
// Complete from poll number `from` on.
struct Barrier {
  std::uint64_t from;
  mutable std::uint64_t polls = 0;
  bool operator()() const { return polls++ >= from; }
};
constexpr std::uint64_t kNever = ~std::uint64_t{0};

}  // namespace

int main() {
  {  // complete at once, and after a while
    const Clock c{1000, kNever, 0};
    EXPECT(q3x::wait_in_time(Barrier{0}, c, kLimit, kPolls));
    EXPECT(q3x::wait_in_time(Barrier{150000}, c, kLimit, kPolls));  // 150 ms
  }
  // switched off the GPU for a second between a poll that failed and the reading of the clock; the barrier is complete by the
  // next poll, or needs another millisecond
  EXPECT(q3x::wait_in_time(Barrier{1}, Clock{1000, 1, 1000 * kMs}, kLimit, kPolls));
  EXPECT(q3x::wait_in_time(Barrier{1000}, Clock{1000, 1, 1000 * kMs}, kLimit, kPolls));
  EXPECT(q3x::wait_in_time(Barrier{70}, Clock{1000, 50, 1000 * kMs}, kLimit, kPolls));
  {  // never complete: the bound holds, with and without time away, and where every poll takes long
    const Clock c{1000, kNever, 0}, away{1000, 100, 5000 * kMs}, slow{10 * kMs, kNever, 0};
    EXPECT(!q3x::wait_in_time(Barrier{kNever}, c, kLimit, kPolls));
    EXPECT(c.now >= kLimit && c.now < kLimit + 2 * kMs);
    EXPECT(!q3x::wait_in_time(Barrier{kNever}, away, kLimit, kPolls));
    EXPECT(away.now >= kLimit + 4999 * kMs && away.now < kLimit + 5002 * kMs);
    EXPECT(!q3x::wait_in_time(Barrier{kNever}, slow, kLimit, kPolls));
    EXPECT(slow.readings <= 203);
  }
  {  // a clock that stands still: the polls are counted too
    const Clock c{0, kNever, 0};
    const Barrier b{kNever};
    EXPECT(!q3x::wait_in_time(b, c, kLimit, 1000));
    EXPECT(b.polls == 1000);
  }
  if (failures == 0) std::printf("bounded wait tests passed\n");
  return failures == 0 ? 0 : 1;
}
