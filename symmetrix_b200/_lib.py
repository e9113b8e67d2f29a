"""ctypes binding of ``libsymmetrix_b200.so`` (the C ABI declared in ``include/symmetrix_b200.h``).

There is deliberately no fallback: if the shared library is missing, or no CUDA device is
usable, creating an evaluator raises.
"""
from __future__ import annotations

import ctypes
from pathlib import Path

PKG = Path(__file__).resolve().parent
LIB_PATH = PKG / "libsymmetrix_b200.so"

SMX_HOST, SMX_DEVICE = 0, 1
SMX_FP32, SMX_FP64 = 32, 64
SMX_OK, SMX_ERR_INVALID_ARGUMENT, SMX_ERR_MODEL, SMX_ERR_CUDA, SMX_ERR_UNSUPPORTED, SMX_ERR_NO_DEVICE = range(6)

# every symbol the header declares (checked by the CPU test-suite against the built library)
EXPORTED_SYMBOLS = [
    "smx_create", "smx_destroy", "smx_last_error", "smx_info", "smx_atomic_numbers", "smx_atomic_energies",
    "smx_compute", "smx_begin", "smx_stage", "smx_get_array", "smx_set_array", "smx_reduce_forces",
    "smx_last_device_ms", "smx_launch_count", "smx_build_neighbors", "smx_evaluate", "smx_get_edges", "smx_compute_current",
    "smx_timer_start", "smx_timer_stop", "smx_set_profiling", "smx_stage_time", "smx_measure_fma_peak", "smx_measure_row_stream", "smx_validate_inputs",
    "smx_energy_virial_noalloc", "smx_sync", "smx_set_stream", "smx_restrict_nodes", "smx_set_active_nodes", "smx_resize_rows", "smx_device_ptr",
    "smx_halo_pack", "smx_halo_unpack", "smx_halo_unpack_add", "smx_halo_cache_lists", "smx_atom_forces", "smx_active_counts", "smx_debug_expire_waits",
    "smx_comm_unique_id", "smx_comm_init", "smx_comm_destroy", "smx_halo_exchange", "smx_allreduce_sum", "smx_model_digest",
    "smx_set_adapters", "smx_assign_adapters", "smx_adapter_gradients", "smx_route_plan_bytes", "smx_route_plan", "smx_route_dispatch", "smx_route_combine", "smx_route_combine_backward",
    "smx_adapter_tiles_bytes", "smx_adapter_prepare", "smx_adapter_hidden_elements", "smx_adapter_workspace_bytes", "smx_adapter_forward", "smx_adapter_backward",
]
ROUTE_MAX_GROUPS, ROUTE_MAX_SLOTS = 1024, 64
ADAPTER_MAX_RANK, ADAPTER_MAX_DEGREES = 64, 8
ADAPTER_SHARED, ADAPTER_MATRICES = 1, 2


class ModelInfo(ctypes.Structure):
    _fields_ = [
        ("num_elements", ctypes.c_int), ("num_channels", ctypes.c_int), ("r_cut", ctypes.c_double),
        ("l_max", ctypes.c_int), ("num_lm", ctypes.c_int), ("L_max", ctypes.c_int), ("num_LM", ctypes.c_int),
        ("num_paths", ctypes.c_int), ("num_lelm1lm2", ctypes.c_int), ("num_lme", ctypes.c_int),
        ("has_zbl", ctypes.c_int), ("precision", ctypes.c_int), ("device", ctypes.c_int),
        ("num_interactions", ctypes.c_int),
    ]


class AdapterDegree(ctypes.Structure):
    _fields_ = [("components", ctypes.c_int), ("in_channels", ctypes.c_int), ("out_channels", ctypes.c_int),
                ("shared", ctypes.c_void_p), ("down", ctypes.c_void_p), ("up", ctypes.c_void_p),
                ("grad_down", ctypes.c_void_p), ("grad_up", ctypes.c_void_p)]


class AdapterCall(ctypes.Structure):
    _fields_ = [("precision", ctypes.c_int), ("num_degrees", ctypes.c_int), ("num_groups", ctypes.c_int), ("rank", ctypes.c_int),
                ("slots", ctypes.c_int), ("num_rows", ctypes.c_long), ("degrees", AdapterDegree * ADAPTER_MAX_DEGREES), ("tiles", ctypes.c_void_p),
                ("order", ctypes.c_void_p), ("position", ctypes.c_void_p), ("offsets", ctypes.c_void_p), ("weights", ctypes.c_void_p),
                ("x", ctypes.c_void_p), ("x_stride", ctypes.c_long), ("y", ctypes.c_void_p), ("y_stride", ctypes.c_long),
                ("grad_y", ctypes.c_void_p), ("grad_y_stride", ctypes.c_long), ("grad_x", ctypes.c_void_p), ("grad_x_stride", ctypes.c_long),
                ("grad_weights", ctypes.c_void_p), ("hidden", ctypes.c_void_p), ("workspace", ctypes.c_void_p),
                ("workspace_bytes", ctypes.c_long), ("stream", ctypes.c_void_p), ("status", ctypes.c_void_p)]


_lib = None


def load():
    """Load the shared library (once) and declare the argument types of every entry point."""
    global _lib
    if _lib is not None:
        return _lib
    if not LIB_PATH.is_file():
        raise RuntimeError(
            f"{LIB_PATH} is missing: build it with `python -m symmetrix_b200.build` (there is no CPU fallback)")
    lib = ctypes.CDLL(str(LIB_PATH))
    vp, ip, dp, lp = ctypes.c_void_p, ctypes.c_void_p, ctypes.c_void_p, ctypes.POINTER(ctypes.c_long)
    lib.smx_create.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ctypes.POINTER(vp)]
    lib.smx_destroy.argtypes = [vp]
    lib.smx_destroy.restype = None
    lib.smx_last_error.argtypes = [vp]
    lib.smx_last_error.restype = ctypes.c_char_p
    lib.smx_info.argtypes = [vp, ctypes.POINTER(ModelInfo)]
    lib.smx_atomic_numbers.argtypes = [vp, ip, ctypes.c_int]
    lib.smx_atomic_energies.argtypes = [vp, dp, ctypes.c_int]
    edge_args = [vp, ctypes.c_int, ip, ip, ip, ip, dp, dp, ctypes.c_long, ctypes.c_int]
    lib.smx_compute.argtypes = edge_args
    lib.smx_begin.argtypes = edge_args
    lib.smx_stage.argtypes = [vp, ctypes.c_char_p, ctypes.c_int, ctypes.c_int]
    lib.smx_get_array.argtypes = [vp, ctypes.c_char_p, dp, ctypes.c_long, lp, ctypes.c_int]
    lib.smx_set_array.argtypes = [vp, ctypes.c_char_p, dp, ctypes.c_long, ctypes.c_int]
    lib.smx_reduce_forces.argtypes = [vp, ctypes.c_int, dp, dp, dp, ctypes.c_int]
    lib.smx_last_device_ms.argtypes = [vp, ctypes.POINTER(ctypes.c_double)]
    lib.smx_launch_count.argtypes = [vp]
    lib.smx_launch_count.restype = ctypes.c_long
    lib.smx_build_neighbors.argtypes = [vp, ctypes.c_int, dp, ip, dp, ip, ctypes.c_double, lp, ctypes.c_int]
    lib.smx_evaluate.argtypes = [vp, ctypes.c_int, dp, ip, dp, ip, ctypes.c_double, dp, dp, dp, dp, lp]
    lib.smx_get_edges.argtypes = [vp, ip, ip, ip, ip, dp, dp, ctypes.c_int]
    lib.smx_compute_current.argtypes = [vp]
    lib.smx_timer_start.argtypes = [vp]
    lib.smx_timer_stop.argtypes = [vp, ctypes.POINTER(ctypes.c_double)]
    lib.smx_set_profiling.argtypes = [vp, ctypes.c_int]
    lib.smx_stage_time.argtypes = [vp, ctypes.c_int, ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(ctypes.c_double)]
    lib.smx_measure_fma_peak.argtypes = [ctypes.c_int, ctypes.c_int, ctypes.POINTER(ctypes.c_double)]
    lib.smx_measure_row_stream.argtypes = [ctypes.c_void_p, ctypes.c_int, ctypes.POINTER(ctypes.c_double), ctypes.POINTER(ctypes.c_double)]
    lib.smx_validate_inputs.argtypes = [vp, ctypes.c_int, lp, lp]
    lib.smx_sync.argtypes = [vp]
    lib.smx_set_stream.argtypes = [vp, vp, ctypes.c_int]
    lib.smx_restrict_nodes.argtypes = [vp, ctypes.c_int, lp]
    lib.smx_set_active_nodes.argtypes = [vp, ctypes.c_int, lp]
    lib.smx_resize_rows.argtypes = [vp, ctypes.c_char_p, ctypes.c_int]
    lib.smx_device_ptr.argtypes = [vp, ctypes.c_char_p, ctypes.POINTER(ctypes.c_void_p), lp, ctypes.POINTER(ctypes.c_int)]
    lib.smx_halo_pack.argtypes = [vp, ctypes.c_char_p, ip, ctypes.c_int, vp]
    lib.smx_halo_unpack.argtypes = [vp, ctypes.c_char_p, ip, ctypes.c_int, vp]
    lib.smx_halo_unpack_add.argtypes = [vp, ctypes.c_char_p, ip, ctypes.c_int, vp]
    lib.smx_atom_forces.argtypes = [vp, ctypes.c_int]
    lib.smx_active_counts.argtypes = [vp, ctypes.POINTER(ctypes.c_int), lp, ctypes.POINTER(ctypes.c_int)]
    lib.smx_debug_expire_waits.argtypes = [vp, ctypes.c_int]
    lib.smx_halo_cache_lists.argtypes = [vp, ctypes.c_int]
    lib.smx_comm_unique_id.argtypes = [vp, ctypes.c_int]
    lib.smx_comm_init.argtypes = [vp, vp, ctypes.c_int, ctypes.c_int, ctypes.c_int]
    lib.smx_comm_destroy.argtypes = [vp]
    lib.smx_halo_exchange.argtypes = [vp, ctypes.c_char_p, ctypes.c_int, ctypes.c_int, ip, vp, ip, vp, ip]
    lib.smx_allreduce_sum.argtypes = [vp, dp, ctypes.c_int]
    lib.smx_model_digest.argtypes = [ctypes.c_char_p, ctypes.c_int, ctypes.POINTER(ctypes.c_ulonglong), ctypes.POINTER(ctypes.c_int)]
    lib.smx_energy_virial_noalloc.argtypes = [dp, ctypes.c_int, dp, dp, ctypes.c_long, dp, vp, ctypes.c_char_p, ctypes.c_int]
    lib.smx_set_adapters.argtypes = [vp, ctypes.c_char_p, ctypes.c_int, ctypes.c_int, dp, ctypes.c_long, dp, ctypes.c_long]
    lib.smx_assign_adapters.argtypes = [vp, ctypes.c_int, ctypes.c_int, ip, dp]
    lib.smx_adapter_gradients.argtypes = [vp, ctypes.c_char_p, dp, dp, dp]
    cl, ci, err = ctypes.c_long, ctypes.c_int, [ctypes.c_char_p, ctypes.c_int]
    lib.smx_route_plan_bytes.argtypes = [cl, ci, ci]
    lib.smx_route_plan_bytes.restype = cl
    lib.smx_route_plan.argtypes = [ip, cl, ci, ci, ip, ip, ip, vp, cl, vp, *err]
    lib.smx_route_dispatch.argtypes = [ci, vp, cl, cl, ci, cl, ip, ip, ci, vp, ci, vp, *err]
    lib.smx_route_combine.argtypes = [ci, vp, ip, cl, ci, cl, vp, vp, cl, vp, cl, vp, *err]
    lib.smx_route_combine_backward.argtypes = [ci, vp, cl, vp, ip, ip, ci, cl, ci, cl, vp, vp, vp, ci, vp, *err]
    call = ctypes.POINTER(AdapterCall)
    lib.smx_adapter_tiles_bytes.argtypes = [call]
    lib.smx_adapter_tiles_bytes.restype = cl
    lib.smx_adapter_prepare.argtypes = [call, ci, *err]
    lib.smx_adapter_hidden_elements.argtypes = [call]
    lib.smx_adapter_hidden_elements.restype = cl
    lib.smx_adapter_workspace_bytes.argtypes = [call, ci]
    lib.smx_adapter_workspace_bytes.restype = cl
    lib.smx_adapter_forward.argtypes = [call, *err]
    lib.smx_adapter_backward.argtypes = [call, *err]
    _lib = lib
    return lib
