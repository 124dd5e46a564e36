#include "nnx_heldtile.h"

namespace nnx {

void held_units_f16(const HeldAttention& h, const HeldPlan& p, hipStream_t st) {
  held_units<f16>(h, p, st);
}

}  // namespace nnx
