// attn_tile_f16_64.cu -- attn_tile_kernel for f16, head sizes up to 64.
#include "attn_tile.cuh"

namespace mgc {
namespace at {
void launch_tile_f16_64(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TileCall& t, cudaStream_t st) {
    dispatch_mode<false, 64>(mq, mk, mv, t, st);
}
}  // namespace at
}  // namespace mgc
