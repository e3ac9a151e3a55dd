// The clipped policy loss for f16 logits (see policy_loss.hpp).
#include "policy_loss.hpp"

using namespace mxh;

MXH_POLICY_LOSS_BOTH(f16_t, f16)
