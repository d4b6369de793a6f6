// The norm of many gradients together, and the gradients scaled by it.
#pragma once
#include "../../include/hetuctr_hip.h"
#include "common.h"

namespace hctr {

// The entry points of the C ABI behind their guard
void gradient_norm(const hctr_clip_args &a, bool clip);
size_t gradient_workspace(const hctr_clip_args &a);

} // namespace hctr
