// Host-side entry points of the embeddings (smx_embedding_*). All work is issued on the given stream of the current device; nothing allocates,
// nothing waits. Argument errors and launch failures throw (common.cuh).
#pragma once

#include <cuda_runtime.h>

#include <cstddef>

#include "../../include/symmetrix_b200.h"

namespace smx {

size_t embedding_plan_bytes(long num_rows, int slots, int table_rows);
void embedding_plan(const int* ids, long num_rows, int slots, int table_rows, int* order, int* tokens, void* workspace, size_t workspace_bytes,
                    cudaStream_t stream);
template <typename T>
void embedding_forward(const T* table, long table_stride, int table_rows, const int* ids, long num_rows, int slots, long width, const T* weights,
                       double scale, T* y, long y_stride, cudaStream_t stream);
template <typename T>
size_t embedding_backward_bytes(long num_rows, int slots, long width);
template <typename T>
void embedding_backward(const T* grad_y, long grad_y_stride, const T* table, long table_stride, int table_rows, const int* order, const int* tokens,
                        long num_rows, int slots, long width, const T* weights, double scale, T* grad_table, T* grad_weights, void* workspace,
                        size_t workspace_bytes, cudaStream_t stream);

}  // namespace smx
