// Host-side entry points of the norm and the clipping of gradients (smx_gradient_*). All work is issued on the given stream of the
// current device; nothing allocates, nothing waits. Argument errors and launch failures throw (common.cuh).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

#include "../../include/symmetrix_b200.h"

namespace smx {

size_t gradient_workspace_bytes(const smx_gradient* list, int count);
// `clip`: also scales; otherwise only the norm.
void gradient_norm_clip(const smx_gradient* list, int count, bool clip, double max_norm, double* norm, void* workspace, size_t workspace_bytes,
                        cudaStream_t stream);

}  // namespace smx
