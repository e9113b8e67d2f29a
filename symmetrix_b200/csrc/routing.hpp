// Host-side entry points of the row routing and of the linears with low-rank adapters, shared by the extern "C" layer and the
// evaluator. All work is issued on the given stream of the current device; nothing allocates, nothing waits. Argument errors and launch
// failures throw (common.cuh).
#pragma once

#include <initializer_list>
#include <cuda_runtime.h>

#include <atomic>

#include "../../include/symmetrix_b200.h"

namespace smx {

// Kernels that this thread launched here and in the files of the operators that include this one.
extern thread_local long operator_launches;

// SMs of the current device; and tables of devices on which a kernel's attributes have been set, which is done once on each.
int sm_count();
bool first_on_device(std::atomic<bool> (&done)[64]);
void mark_on_device(std::atomic<bool> (&done)[64]);

size_t route_plan_bytes(long num_rows, int slots, int num_groups);
void route_plan(const int* ids, long num_rows, int slots, int num_groups, int* order, int* position, int* offsets, void* workspace,
                size_t workspace_bytes, cudaStream_t stream);
// Refuses pointers that do not start on a multiple of `bytes` (kernels would fault on them).
void check_pointers(const char* what, size_t bytes, std::initializer_list<const void*> pointers);
// The plan slot by slot: places[s * num_rows ..] are the sorted positions of slot s's pairs, ascending, so grouped, empty ones last;
// slot_offsets[s * (num_groups + 1) + g] is where group g begins among them. A row is in every slot's list once.
size_t route_slots_bytes(long num_rows, int slots);
void route_slots(const int* order, long num_rows, int slots, const int* offsets, int num_groups, int* places, int* slot_offsets, void* workspace,
                 cudaStream_t stream);
// Pairs by token, equal ones in the order of the list, those without one (outside 0 .. table_rows - 1) last: order[p] is the p-th, names[p] its token
// (table_rows: none). Fewer than 2^20 table rows; the caller has checked the sizes.
size_t token_sort_bytes(long pairs, int table_rows);
void token_sort(const int* ids, long pairs, int table_rows, int* order, int* names, void* workspace, cudaStream_t stream);
template <typename T>
void route_dispatch(const T* x, long x_stride, long num_rows, int slots, long width, const int* position, const int* offsets, int num_groups,
                    T* rows, bool zero_tail, cudaStream_t stream);
template <typename T>
void route_combine(const T* rows, const int* position, long num_rows, int slots, long width, const T* weights, const T* base, long base_stride,
                   T* y, long y_stride, cudaStream_t stream);
template <typename T>
void route_combine_backward(const T* grad_y, long grad_y_stride, const T* rows, const int* position, const int* offsets, int num_groups,
                            long num_rows, int slots, long width, const T* weights, T* grad_rows, T* grad_weights, bool zero_tail,
                            cudaStream_t stream);

}  // namespace smx
