// The extern "C" entry points declared in include/symmetrix_b200.h: argument checks, exception -> status code,
// and dispatch to the evaluator of the handle's precision.
#include <cuda_runtime.h>

#include <cstdio>
#include <cstring>
#include <memory>
#include <stdexcept>
#include <string>
#include <type_traits>

#include "../../include/symmetrix_b200.h"
#include "adapters.hpp"
#include "embedding.hpp"
#include "gradients.hpp"
#include "grouped.hpp"
#include "common.cuh"
#include "evaluator_base.hpp"
#include "model_cache.hpp"
#include "nccl_transport.hpp"
#include "routing.hpp"

// =================================================================================================
// extern "C" entry points
// =================================================================================================
struct smx_evaluator {
    std::unique_ptr<smx::EvaluatorBase> impl;
};

namespace {
thread_local std::string g_create_error;

template <typename Fn>
int guarded(smx_handle h, Fn&& fn) {
    if (!h || !h->impl) return SMX_ERR_INVALID_ARGUMENT;
    try {
        fn(*h->impl);
        return SMX_OK;
    } catch (const smx::ArgError& e) {
        h->impl->last_error = e.what();
        return SMX_ERR_INVALID_ARGUMENT;
    } catch (const smx::UnsupportedError& e) {
        h->impl->last_error = e.what();
        return SMX_ERR_UNSUPPORTED;
    } catch (const smx::CudaError& e) {
        h->impl->last_error = e.what();
        return SMX_ERR_CUDA;
    } catch (const std::exception& e) {
        h->impl->last_error = e.what();
        return SMX_ERR_INVALID_ARGUMENT;
    }
}

// Calls without an evaluator: the message goes to the caller's buffer.
template <typename Fn>
int guarded_free(char* errbuf, int errbuf_len, Fn&& fn) {
    auto fail = [&](int status, const char* what) {
        if (errbuf && errbuf_len > 0) std::snprintf(errbuf, static_cast<size_t>(errbuf_len), "%s", what);
        return status;
    };
    try {
        fn();
        return SMX_OK;
    } catch (const smx::ArgError& e) { return fail(SMX_ERR_INVALID_ARGUMENT, e.what());
    } catch (const smx::CudaError& e) { return fail(SMX_ERR_CUDA, e.what());
    } catch (const std::exception& e) { return fail(SMX_ERR_INVALID_ARGUMENT, e.what()); }
}
template <typename Fn>
long size_or_refusal(Fn&& fn) {
    try {
        return static_cast<long>(fn());
    } catch (const std::exception&) { return -1; }
}
// Calls fn with a null pointer of the precision's type.
template <typename Fn>
void with_precision(int precision, const char* what, Fn&& fn) {
    if (precision == SMX_FP32) fn(static_cast<float*>(nullptr));
    else if (precision == SMX_FP64) fn(static_cast<double*>(nullptr));
    else throw smx::ArgError(std::string(what) + ": precision must be 32 or 64");
}
}  // namespace

extern "C" {

int smx_create(const char* json_path, int precision, int device, smx_handle* out) {
    if (!out) return SMX_ERR_INVALID_ARGUMENT;
    *out = nullptr;
    try {
        if (!json_path) throw smx::ArgError("smx_create: null path");
        if (precision != SMX_FP32 && precision != SMX_FP64) throw smx::ArgError("smx_create: precision must be 32 or 64");
        // the model is read and validated first, so a bad file is reported as such on any machine
        smx::HostModel m = smx::load_model_cached(json_path);
        int count = 0;
        if (cudaGetDeviceCount(&count) != cudaSuccess || count == 0) {
            cudaGetLastError();
            g_create_error = "no CUDA device available: this library has no CPU path";
            return SMX_ERR_NO_DEVICE;
        }
        if (device < 0 || device >= count) throw smx::ArgError("smx_create: device ordinal out of range");
        auto h = std::make_unique<smx_evaluator>();
        if (precision == SMX_FP32) h->impl = smx::make_evaluator_f32(std::move(m), device);
        else h->impl = smx::make_evaluator_f64(std::move(m), device);
        *out = h.release();
        return SMX_OK;
    } catch (const smx::ArgError& e) { g_create_error = e.what(); return SMX_ERR_INVALID_ARGUMENT;
    } catch (const smx::UnsupportedError& e) { g_create_error = e.what(); return SMX_ERR_UNSUPPORTED;
    } catch (const smx::CudaError& e) { g_create_error = e.what(); return SMX_ERR_CUDA;
    } catch (const std::exception& e) { g_create_error = e.what(); return SMX_ERR_MODEL; }  // JsonError, ModelError, I/O
}

void smx_destroy(smx_handle h) { delete h; }

const char* smx_last_error(smx_handle h) {
    if (!h || !h->impl) return g_create_error.c_str();
    return h->impl->last_error.c_str();
}

int smx_info(smx_handle h, smx_model_info* info) {
    if (!info) return SMX_ERR_INVALID_ARGUMENT;
    return guarded(h, [&](smx::EvaluatorBase& e) {
        const smx::HostModel& m = e.model;
        info->num_elements = m.num_elements; info->num_channels = m.K; info->r_cut = m.r_cut;
        info->l_max = m.l_max; info->num_lm = m.num_lm; info->L_max = m.L_max; info->num_LM = m.num_LM;
        info->num_paths = m.tp.P; info->num_lelm1lm2 = m.tp.T; info->num_lme = m.tp.Q;
        info->num_interactions = m.num_interactions;
        info->has_zbl = m.has_zbl ? 1 : 0; info->precision = e.precision; info->device = e.device;
    });
}

int smx_atomic_numbers(smx_handle h, int* out, int cap) {
    if (!h || !h->impl) return -1;
    const auto& v = h->impl->model.atomic_numbers;
    for (int i = 0; i < static_cast<int>(v.size()) && i < cap && out; ++i) out[i] = v[i];
    return static_cast<int>(v.size());
}
int smx_atomic_energies(smx_handle h, double* out, int cap) {
    if (!h || !h->impl) return -1;
    const auto& v = h->impl->model.atomic_energies;
    for (int i = 0; i < static_cast<int>(v.size()) && i < cap && out; ++i) out[i] = v[i];
    return static_cast<int>(v.size());
}

int smx_begin(smx_handle h, int num_nodes, const int* node_types, const int* num_neigh, const int* neigh_indices,
              const int* neigh_types, const double* xyz, const double* r, long num_edges, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        e.begin(num_nodes, node_types, num_neigh, neigh_indices, neigh_types, xyz, r, num_edges, mem_space);
    });
}

int smx_compute(smx_handle h, int num_nodes, const int* node_types, const int* num_neigh, const int* neigh_indices,
                const int* neigh_types, const double* xyz, const double* r, long num_edges, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        e.begin(num_nodes, node_types, num_neigh, neigh_indices, neigh_types, xyz, r, num_edges, mem_space);
        e.compute_all();
    });
}

int smx_compute_current(smx_handle h) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.compute_all(); });
}

int smx_stage(smx_handle h, const char* name, int zero_dxyz, int zero_H1_adj) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_stage: null name");
        e.stage(name, zero_dxyz != 0, zero_H1_adj != 0);
    });
}

int smx_get_array(smx_handle h, const char* name, double* dst, long cap, long* n, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_get_array: null name");
        const long count = e.get_array(name, dst, cap, mem_space);
        if (n) *n = count;
    });
}

int smx_set_array(smx_handle h, const char* name, const double* src, long n, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_set_array: null name");
        e.set_array(name, src, n, mem_space);
    });
}

int smx_reduce_forces(smx_handle h, int num_rows, double* atom_forces, double* virial, double* energy, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.reduce_forces(num_rows, atom_forces, virial, energy, mem_space); });
}

int smx_atom_forces(smx_handle h, int num_rows) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.atom_forces(num_rows); });
}

int smx_halo_pack(smx_handle h, const char* name, const int* rows, int n, void* dst) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_halo_pack: null name");
        e.halo_pack(name, rows, n, dst);
    });
}
int smx_halo_unpack(smx_handle h, const char* name, const int* rows, int n, const void* src) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_halo_unpack: null name");
        e.halo_unpack(name, rows, n, src, false);
    });
}
int smx_halo_unpack_add(smx_handle h, const char* name, const int* rows, int n, const void* src) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_halo_unpack_add: null name");
        e.halo_unpack(name, rows, n, src, true);
    });
}
int smx_model_digest(const char* json_path, int use_cache, unsigned long long* digest, int* from_cache) {
    try {
        if (!json_path || !digest) throw smx::ArgError("smx_model_digest: null argument");
        bool hit = false;
        smx::HostModel m = use_cache ? smx::load_model_cached(json_path, &hit) : smx::load_model_file(json_path);
        *digest = smx::model_digest(m);
        if (from_cache) *from_cache = hit ? 1 : 0;
        return SMX_OK;
    } catch (const smx::ArgError& e) { g_create_error = e.what(); return SMX_ERR_INVALID_ARGUMENT;
    } catch (const smx::UnsupportedError& e) { g_create_error = e.what(); return SMX_ERR_UNSUPPORTED;
    } catch (const std::exception& e) { g_create_error = e.what(); return SMX_ERR_MODEL; }
}

int smx_comm_unique_id(void* id, int id_bytes) {
    try {
        if (!id || id_bytes != static_cast<int>(sizeof(smx::NcclApi::UniqueId))) throw smx::ArgError("smx_comm_unique_id: the id buffer must hold 128 bytes");
        const smx::NcclApi& nccl = smx::NcclApi::get();
        smx::NcclApi::UniqueId uid;
        nccl.check(nccl.GetUniqueId(&uid), "ncclGetUniqueId");
        std::memcpy(id, &uid, sizeof(uid));
        return SMX_OK;
    } catch (const smx::ArgError& e) { g_create_error = e.what(); return SMX_ERR_INVALID_ARGUMENT;
    } catch (const std::exception& e) { g_create_error = e.what(); return SMX_ERR_CUDA; }
}
int smx_comm_init(smx_handle h, const void* id, int id_bytes, int num_ranks, int rank) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.comm_init(id, id_bytes, num_ranks, rank); });
}
int smx_comm_destroy(smx_handle h) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.comm_destroy(); });
}
int smx_halo_exchange(smx_handle h, const char* name, int add, int num_peers, const int* peers, const int* const* send_rows,
                      const int* send_counts, const int* const* recv_rows, const int* recv_counts) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_halo_exchange: null name");
        e.halo_exchange(name, add != 0, num_peers, peers, send_rows, send_counts, recv_rows, recv_counts);
    });
}
int smx_allreduce_sum(smx_handle h, double* values, int n) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.allreduce_sum(values, n); });
}
int smx_active_counts(smx_handle h, int* num_nodes, long* num_edges, int* built_nodes) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.active_counts(num_nodes, num_edges, built_nodes); });
}
int smx_halo_cache_lists(smx_handle h, int enable) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.halo_cache_lists(enable); });
}
int smx_debug_expire_waits(smx_handle h, int polls) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.expire_waits(polls); });
}

int smx_last_device_ms(smx_handle h, double* ms) {
    return guarded(h, [&](smx::EvaluatorBase& e) { if (ms) *ms = e.last_ms; });
}

long smx_launch_count(smx_handle h) { return (h && h->impl) ? h->impl->launches : -1; }

int smx_sync(smx_handle h) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.sync(); });
}
int smx_set_stream(smx_handle h, void* stream, int external) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.set_stream(stream, external != 0); });
}
int smx_restrict_nodes(smx_handle h, int num_nodes, long* num_edges) {
    return guarded(h, [&](smx::EvaluatorBase& e) { const long n = e.restrict_nodes(num_nodes, false); if (num_edges) *num_edges = n; });
}

int smx_set_active_nodes(smx_handle h, int num_nodes, long* num_edges) {
    return guarded(h, [&](smx::EvaluatorBase& e) { const long n = e.restrict_nodes(num_nodes, true); if (num_edges) *num_edges = n; });
}
int smx_resize_rows(smx_handle h, const char* name, int rows) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name) throw smx::ArgError("smx_resize_rows: null name");
        e.resize_rows(name, rows);
    });
}
int smx_device_ptr(smx_handle h, const char* name, void** ptr, long* count, int* elem_bytes) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!name || !ptr) throw smx::ArgError("smx_device_ptr: null argument");
        *ptr = e.device_ptr(name, count, elem_bytes);
    });
}
int smx_timer_start(smx_handle h) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.timer_start(); });
}
int smx_timer_stop(smx_handle h, double* ms) {
    return guarded(h, [&](smx::EvaluatorBase& e) { const double t = e.timer_stop(); if (ms) *ms = t; });
}
int smx_set_profiling(smx_handle h, int enabled) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.profiling = enabled != 0; });
}
int smx_stage_time(smx_handle h, int index, char* name, int name_cap, double* ms) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (index < 0 || index >= static_cast<int>(e.stage_ms.size())) throw smx::ArgError("smx_stage_time: index out of range");
        if (name && name_cap > 0) {
            std::strncpy(name, e.stage_ms[index].first.c_str(), name_cap - 1);
            name[name_cap - 1] = 0;
        }
        if (ms) *ms = e.stage_ms[index].second;
    });
}

int smx_measure_fma_peak(int precision, int device, double* tflops) {
    try {
        if (!tflops) throw smx::ArgError("null output");
        *tflops = precision == SMX_FP32 ? smx::measure_fma_peak_f32(device) : smx::measure_fma_peak_f64(device);
        return SMX_OK;
    } catch (const std::exception& e) {
        g_create_error = e.what();
        return SMX_ERR_CUDA;
    }
}

int smx_measure_row_stream(smx_handle h, int layer, double* ms, double* bytes) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.measure_row_stream(layer, ms, bytes); });
}

int smx_validate_inputs(smx_handle h, int feature_rows, long* counts, long* total) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        const long n = e.validate_inputs(feature_rows, counts);
        if (total) *total = n;
        if (n != 0) throw smx::ArgError("the edge arrays hold " + std::to_string(n) + " out-of-range or inconsistent entries");
    });
}

int smx_build_neighbors(smx_handle h, int num_atoms, const double* positions, const int* types, const double* cell,
                        const int* pbc, double r_cut, long* num_edges, int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        const long n = e.build_neighbors(num_atoms, positions, types, cell, pbc, r_cut, mem_space);
        if (num_edges) *num_edges = n;
    });
}

int smx_evaluate(smx_handle h, int num_atoms, const double* positions, const int* types, const double* cell, const int* pbc, double r_cut,
                 double* forces, double* energies, double* virial, double* energy, long* num_edges) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        const long n = e.evaluate(num_atoms, positions, types, cell, pbc, r_cut, forces, energies, virial, energy);
        if (num_edges) *num_edges = n;
    });
}

int smx_get_edges(smx_handle h, int* num_neigh, int* neigh_indices, int* neigh_types, int* shifts, double* xyz, double* r,
                  int mem_space) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.get_edges(num_neigh, neigh_indices, neigh_types, shifts, xyz, r, mem_space); });
}

int smx_set_adapters(smx_handle h, const char* linear, int num_adapters, int rank, const double* down, long down_count, const double* up, long up_count) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!linear) throw smx::ArgError("smx_set_adapters: null name");
        e.set_adapters(linear, num_adapters, rank, down, down_count, up, up_count);
    });
}
int smx_assign_adapters(smx_handle h, int num_nodes, int slots, const int* ids, const double* weights) {
    return guarded(h, [&](smx::EvaluatorBase& e) { e.assign_adapters(num_nodes, slots, ids, weights); });
}
int smx_adapter_gradients(smx_handle h, const char* linear, double* grad_down, double* grad_up, double* grad_weights) {
    return guarded(h, [&](smx::EvaluatorBase& e) {
        if (!linear) throw smx::ArgError("smx_adapter_gradients: null name");
        e.adapter_gradients(linear, grad_down, grad_up, grad_weights);
    });
}
long smx_route_plan_bytes(long num_rows, int slots, int num_groups) {
    return size_or_refusal([&] { return smx::route_plan_bytes(num_rows, slots, num_groups); });
}
int smx_route_plan(const int* ids, long num_rows, int slots, int num_groups, int* order, int* position, int* offsets, void* workspace,
                   long workspace_bytes, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (workspace_bytes < 0) throw smx::ArgError("smx_route_plan: negative workspace size");
        smx::route_plan(ids, num_rows, slots, num_groups, order, position, offsets, workspace, static_cast<size_t>(workspace_bytes),
                        static_cast<cudaStream_t>(stream));
    });
}
int smx_route_dispatch(int precision, const void* x, long x_stride, long num_rows, int slots, long width, const int* position,
                       const int* offsets, int num_groups, void* rows, int zero_tail, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        with_precision(precision, "smx_route_dispatch", [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            smx::route_dispatch<T>(static_cast<const T*>(x), x_stride, num_rows, slots, width, position, offsets, num_groups, static_cast<T*>(rows),
                                   zero_tail != 0, static_cast<cudaStream_t>(stream));
        });
    });
}
int smx_route_combine(int precision, const void* rows, const int* position, long num_rows, int slots, long width, const void* weights,
                      const void* base, long base_stride, void* y, long y_stride, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        with_precision(precision, "smx_route_combine", [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            smx::route_combine<T>(static_cast<const T*>(rows), position, num_rows, slots, width, static_cast<const T*>(weights),
                                  static_cast<const T*>(base), base_stride, static_cast<T*>(y), y_stride, static_cast<cudaStream_t>(stream));
        });
    });
}
int smx_route_combine_backward(int precision, const void* grad_y, long grad_y_stride, const void* rows, const int* position,
                               const int* offsets, int num_groups, long num_rows, int slots, long width, const void* weights,
                               void* grad_rows, void* grad_weights, int zero_tail, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        with_precision(precision, "smx_route_combine_backward", [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            smx::route_combine_backward<T>(static_cast<const T*>(grad_y), grad_y_stride, static_cast<const T*>(rows), position, offsets, num_groups,
                                           num_rows, slots, width, static_cast<const T*>(weights), static_cast<T*>(grad_rows),
                                           static_cast<T*>(grad_weights), zero_tail != 0, static_cast<cudaStream_t>(stream));
        });
    });
}
long smx_adapter_tiles_bytes(const smx_adapter_linear* call) {
    return call ? size_or_refusal([&] { return smx::adapter_tiles_bytes(*call); }) : -1;
}
int smx_adapter_prepare(const smx_adapter_linear* call, int parts, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (!call) throw smx::ArgError("smx_adapter_prepare: null call");
        smx::adapter_prepare(*call, parts);
    });
}
long smx_adapter_hidden_elements(const smx_adapter_linear* call) {
    return call ? size_or_refusal([&] { return smx::adapter_hidden_elements(*call); }) : -1;
}
long smx_adapter_workspace_bytes(const smx_adapter_linear* call, int backward) {
    return call ? size_or_refusal([&] { return smx::adapter_workspace_bytes(*call, backward != 0); }) : -1;
}
int smx_adapter_forward(const smx_adapter_linear* call, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (!call) throw smx::ArgError("smx_adapter_forward: null call");
        smx::adapter_forward(*call);
    });
}
int smx_adapter_backward(const smx_adapter_linear* call, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (!call) throw smx::ArgError("smx_adapter_backward: null call");
        smx::adapter_backward(*call);
    });
}

long smx_grouped_workspace_bytes(const smx_grouped_linear* call, int backward) {
    return call ? size_or_refusal([&] { return smx::grouped_workspace_bytes(*call, backward != 0); }) : -1;
}
int smx_grouped_forward(const smx_grouped_linear* call, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (!call) throw smx::ArgError("smx_grouped_forward: null call");
        smx::grouped_forward(*call);
    });
}
int smx_grouped_backward(const smx_grouped_linear* call, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (!call) throw smx::ArgError("smx_grouped_backward: null call");
        smx::grouped_backward(*call);
    });
}
long smx_embedding_plan_bytes(long num_rows, int slots, int table_rows) {
    return size_or_refusal([&] { return smx::embedding_plan_bytes(num_rows, slots, table_rows); });
}
int smx_embedding_plan(const int* ids, long num_rows, int slots, int table_rows, int* order, int* tokens, void* workspace, long workspace_bytes,
                       void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (workspace_bytes < 0) throw smx::ArgError("smx_embedding_plan: negative workspace size");
        smx::embedding_plan(ids, num_rows, slots, table_rows, order, tokens, workspace, static_cast<size_t>(workspace_bytes), static_cast<cudaStream_t>(stream));
    });
}
int smx_embedding_forward(int precision, const void* table, long table_stride, int table_rows, const int* ids, long num_rows, int slots, long width,
                          const void* weights, double scale, void* y, long y_stride, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        with_precision(precision, "smx_embedding_forward", [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            smx::embedding_forward<T>(static_cast<const T*>(table), table_stride, table_rows, ids, num_rows, slots, width, static_cast<const T*>(weights), scale,
                                      static_cast<T*>(y), y_stride, static_cast<cudaStream_t>(stream));
        });
    });
}
long smx_embedding_backward_bytes(int precision, long num_rows, int slots, long width) {
    return size_or_refusal([&] {
        size_t n = 0;
        with_precision(precision, "smx_embedding_backward", [&](auto* t) { n = smx::embedding_backward_bytes<std::remove_pointer_t<decltype(t)>>(num_rows, slots, width); });
        return n;
    });
}
int smx_embedding_backward(int precision, const void* grad_y, long grad_y_stride, const void* table, long table_stride, int table_rows, const int* order,
                           const int* tokens, long num_rows, int slots, long width, const void* weights, double scale, void* grad_table, void* grad_weights,
                           void* workspace, long workspace_bytes, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (workspace_bytes < 0) throw smx::ArgError("smx_embedding_backward: negative workspace size");
        with_precision(precision, "smx_embedding_backward", [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            smx::embedding_backward<T>(static_cast<const T*>(grad_y), grad_y_stride, static_cast<const T*>(table), table_stride, table_rows, order, tokens, num_rows,
                                       slots, width, static_cast<const T*>(weights), scale, static_cast<T*>(grad_table), static_cast<T*>(grad_weights), workspace,
                                       static_cast<size_t>(workspace_bytes), static_cast<cudaStream_t>(stream));
        });
    });
}
long smx_gradient_workspace_bytes(const smx_gradient* list, int count) {
    return size_or_refusal([&] { return smx::gradient_workspace_bytes(list, count); });
}
int smx_gradient_norm(const smx_gradient* list, int count, double* norm, void* workspace, long workspace_bytes, void* stream, char* errbuf, int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (workspace_bytes < 0) throw smx::ArgError("smx_gradient_norm: negative workspace size");
        smx::gradient_norm_clip(list, count, false, 0.0, norm, workspace, static_cast<size_t>(workspace_bytes), static_cast<cudaStream_t>(stream));
    });
}
int smx_gradient_clip(const smx_gradient* list, int count, double max_norm, double* norm, void* workspace, long workspace_bytes, void* stream, char* errbuf,
                      int errbuf_len) {
    return guarded_free(errbuf, errbuf_len, [&] {
        if (workspace_bytes < 0) throw smx::ArgError("smx_gradient_clip: negative workspace size");
        smx::gradient_norm_clip(list, count, true, max_norm, norm, workspace, static_cast<size_t>(workspace_bytes), static_cast<cudaStream_t>(stream));
    });
}

}  // extern "C"
