// Host-side entry points of the linears of routed rows (smx_grouped_*). All work is issued on the call's stream of the current device; nothing
// allocates, nothing waits. Errors throw (common.cuh).
#pragma once

#include <cstddef>

#include "../../include/symmetrix_b200.h"

namespace smx {

size_t grouped_workspace_bytes(const smx_grouped_linear& c, bool backward);
void grouped_forward(const smx_grouped_linear& c);
void grouped_backward(const smx_grouped_linear& c);

}  // namespace smx
