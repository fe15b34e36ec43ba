/** @brief The dense products' tiles of bfloat16. @file numkong_amd/csrc/dense_gfx950_bf16.hip */
#include "dense_tiles_gfx950.hpp"

namespace nk_gfx950 {
int launch_tiles_bf16(TileForm const &form, TileArgs const &args, hipStream_t stream) { return launch_tiles_of<__bf16>(form, args, stream); }
} // namespace nk_gfx950
