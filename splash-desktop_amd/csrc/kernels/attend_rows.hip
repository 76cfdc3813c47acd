#include "attend_rows.hpp"

namespace sq::kern {

hipError_t launch_attend_rows(uint32_t tile_rows, uint32_t waves, const AttendArgs &a, hipStream_t stream) {
  return launch_rows(tile_rows, waves, a, stream);
}

}  // namespace sq::kern
