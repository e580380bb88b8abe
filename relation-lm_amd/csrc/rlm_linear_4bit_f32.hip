// Products of many fp32 tokens with 4-bit weights (rlm_linear_4bit_tile.hpp).
#include "rlm_linear_4bit_tile.hpp"

namespace rlm {
namespace linear4 {

hipError_t tile_launch_f32(const LinearParams& p, TileShape shape, int products, int scale_dtype,
                           hipStream_t stream) {
  return launch_tile_type<float>(p, shape, products, scale_dtype, stream);
}

}  // namespace linear4
}  // namespace rlm
