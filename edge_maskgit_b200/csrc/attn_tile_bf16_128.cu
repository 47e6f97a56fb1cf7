// attn_tile_bf16_128.cu -- attn_tile_kernel for bf16, head sizes 65 to 128.
#include "attn_tile.cuh"

namespace mgc {
namespace at {
void launch_tile_bf16_128(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TileCall& t, cudaStream_t st) {
    dispatch_mode<true, 128>(mq, mk, mv, t, st);
}
}  // namespace at
}  // namespace mgc
