// Attention for f16 tensors (see attention.hpp).
#include "attention.hpp"

using namespace mxh;

MXH_ATTENTION(f16_t, f16)
