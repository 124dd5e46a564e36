#include "nnx_heldtile.h"

namespace nnx {

void held_units_bf16(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  held_units<bf16>(h, p, st);
}

}  // namespace nnx
