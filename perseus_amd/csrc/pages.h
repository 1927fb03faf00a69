// Keys in pages: by which entry of its sequence's table a run of rows is found (tiles.h loads them). Nothing here needs a GPU.
#pragma once
#include <cstdint>

namespace pch {
namespace clear {

constexpr int RUN = 16;  // rows that are loaded together, in one page

// The entry of the run that begins `run` rows into tile t of KT keys, of a sequence of len keys (one or more) in pages of 2^log rows;
// a tile begins at a page or lies in one. Runs and tiles past the last key, whose numbers are asked for all the same, take the last
// key's entry: a table need have no more.
template <int KT>
constexpr uint32_t entry_of(int t, int run, int log, int len) {
    const uint32_t at = ((uint32_t)t * KT >> log) + ((uint32_t)run >> log), last = (uint32_t)(len - 1) >> log;
    return at < last ? at : last;
}

}  // namespace clear
}  // namespace pch
