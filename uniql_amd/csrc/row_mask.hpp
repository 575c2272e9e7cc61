// Rows of a short run as bits, plain C++ for the host and the GPU: which of them lie in a range, and which in either of two.
#pragma once

#include <stdint.h>

namespace uniql {

// The rows first .. last - 1 of a run of `rows` (32 at most), whatever the bounds are: none behind the run.
constexpr uint32_t rows_between(int first, int last, int rows) {
    first = first < 0 ? 0 : first;
    last = last > rows ? rows : last;
    return first < last ? (uint32_t)(((1ULL << (last - first)) - 1) << first) : 0u;
}
// (Offsets that fall give ranges which meet: a sum of their masks would carry into rows behind the run.)
constexpr uint32_t rows_of_either(uint32_t a, uint32_t b) { return a | b; }

}  // namespace uniql
