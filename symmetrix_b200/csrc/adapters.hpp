// Host-side entry points of the linears with low-rank adapters (smx_adapter_*), shared by the extern "C" layer and the evaluator. All work
// is issued on the call's stream of the current device; nothing allocates, nothing waits. Errors throw (common.cuh).
#pragma once

#include <cstddef>

#include "../../include/symmetrix_b200.h"

namespace smx {

size_t adapter_tiles_bytes(const smx_adapter_linear& c);
void adapter_prepare(const smx_adapter_linear& c, int parts);
size_t adapter_hidden_elements(const smx_adapter_linear& c);
size_t adapter_workspace_bytes(const smx_adapter_linear& c, bool backward);
// `expire_polls`: test switch, see smx_debug_expire_waits.
void adapter_forward(const smx_adapter_linear& c, int expire_polls = 0);
void adapter_backward(const smx_adapter_linear& c, int expire_polls = 0);

}  // namespace smx
