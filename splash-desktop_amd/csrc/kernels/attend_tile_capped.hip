// Calls with capped scores alone on the wide tile: a translation unit of its own beside attend_tile.hip's, for the build's sake.
#include "attend_tile.hpp"

namespace sq::kern {

hipError_t launch_attend_tile_capped(const CappedArgs &a, hipStream_t stream) { return launch_tile(a, stream); }

}  // namespace sq::kern
