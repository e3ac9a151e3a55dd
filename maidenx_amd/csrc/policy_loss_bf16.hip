// The clipped policy loss for bf16 logits (see policy_loss.hpp).
#include "policy_loss.hpp"

using namespace mxh;

MXH_POLICY_LOSS_BOTH(bf16_t, bf16)
