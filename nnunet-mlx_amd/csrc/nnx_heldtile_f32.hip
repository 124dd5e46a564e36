#include "nnx_heldtile.h"

namespace nnx {

void held_units_f32(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  held_units<float>(h, p, st);
}

}  // namespace nnx
