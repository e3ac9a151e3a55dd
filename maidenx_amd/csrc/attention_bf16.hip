// Attention for bf16 tensors (see attention.hpp).
#include "attention.hpp"

using namespace mxh;

MXH_ATTENTION(bf16_t, bf16)
