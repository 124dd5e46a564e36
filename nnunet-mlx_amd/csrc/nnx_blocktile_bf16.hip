#include "nnx_blocktile.h"

namespace nnx {

void block_partials_bf16(const ChunkArgs& c, bool by_block, int grid, hipStream_t st) {
  block_partials<bf16>(c, by_block, grid, st);
}

}  // namespace nnx
