// wait_limit.h -- iteration limit of the decode kernels' bounded on-chip waits.
#pragma once
#include <stdint.h>

namespace fp8mla {
// try_wait suspends for a hardware-chosen interval per call (about 87 ns on
// B200, so 2^22 calls take about 0.4 s): well beyond the longest legitimate
// wait, which spans a few tiles or one change of unit (tens of microseconds)
// and never a whole call, yet a broken protocol ends in under a second with
// the timeout recorded.
constexpr uint32_t kMaxWaitIters = 1u << 22;
// The same for waits in which every lane of a warp looks: such a try_wait suspends
// the warp for up to 7850 cycles (4.0 us, measured; 140 cycles where one lane looks
// for the others), so 2^16 of them take 0.26 s, and 5 ms if each came back at once.
constexpr uint32_t kMaxWaitLooks = kMaxWaitIters / 64;
}  // namespace fp8mla
