#include "attend_tile.hpp"

namespace sq::kern {

hipError_t launch_attend_tile(const AttendArgs &a, hipStream_t stream) { return launch_tile(a, stream); }

}  // namespace sq::kern
