// Scored calls on tiles of few rows: a translation unit of its own beside attend_rows.hip's, for the build's sake.
#include "attend_rows.hpp"

namespace sq::kern {

hipError_t launch_attend_rows_scored(uint32_t tile_rows, uint32_t waves, const ScoredArgs &a, hipStream_t stream) {
  return launch_rows(tile_rows, waves, a, stream);
}

}  // namespace sq::kern
