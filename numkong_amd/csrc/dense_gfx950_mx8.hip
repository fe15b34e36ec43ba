/** @brief The dense products' tiles of 8-bit floats with scales. @file numkong_amd/csrc/dense_gfx950_mx8.hip */
#include "dense_tiles_gfx950.hpp"

namespace nk_gfx950 {
int launch_tiles_mx8(TileForm const &form, TileArgs const &args, hipStream_t stream) { return launch_tiles_of<Mx8>(form, args, stream); }
} // namespace nk_gfx950
