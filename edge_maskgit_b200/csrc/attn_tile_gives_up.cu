// attn_tile_gives_up.cu -- attn_tile_kernel with a wait that gives up (mgc_selftest_attention_gives_up).
#include "attn_tile.cuh"

namespace mgc {
namespace at {
void launch_tile_gives_up(const CUtensorMap& mq, const CUtensorMap& mk, const CUtensorMap& mv, const TileCall& t, cudaStream_t st) {
    launch_tile<false, 64, TABLE, true>(mq, mk, mv, t, st);
}
}  // namespace at
}  // namespace mgc
