// How many workgroups one launch may have.  No device code: a host compiler takes it as it is.
#pragma once
#include <cstdint>

namespace twm {

// A launch whose workgroups stand in a row is to have fewer than 2^32 threads; half as many leave room for what a caller rounds up.
constexpr uint32_t most_workgroups(uint32_t threads) { return (1u << 31) / threads; }

}  // namespace twm
