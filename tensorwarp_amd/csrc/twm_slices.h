// How rows are shared out among launches.  No device code: a host compiler takes it as it is.
#pragma once
#include <cstdint>

namespace twm {

// A launch whose workgroups stand in a row is to have fewer than 2^32 threads; half as many leave room for what a caller rounds up.
constexpr uint32_t most_workgroups(uint32_t threads) { return (1u << 31) / threads; }

// launch(first, count) for the rows 0 .. rows - 1, at most `most` at a time, up to the first one that fails, whose error is returned.
template <typename F> auto in_slices(uint32_t rows, uint32_t most, F &&launch) -> decltype(launch(0u, 0u))
{
    decltype(launch(0u, 0u)) error{};
    for (uint64_t row = 0; row < rows && error == decltype(error){}; row += most) error = launch((uint32_t)row, rows - row < most ? (uint32_t)(rows - row) : most);
    return error;
}

}  // namespace twm
