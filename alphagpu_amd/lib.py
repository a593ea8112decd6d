"""ctypes binding of libagz.so (include/agz.h)."""
import ctypes as C
import os
import subprocess

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.environ.get("AGZ_LIB_PATH") or os.path.join(_HERE, "libagz.so")   # (AGZ_LIB_PATH: an alternative build of the library, A/B measurements)
CSRC = os.path.join(_HERE, "csrc")
_LIB = None


class LibraryMissing(RuntimeError):
    pass


class AgzError(RuntimeError):
    def __init__(self, code, msg):
        super().__init__(f"libagz error {code}: {msg}")
        self.code = code


class Config(C.Structure):
    _fields_ = [("game", C.c_int32), ("n", C.c_int32), ("nvict", C.c_int32), ("max_games", C.c_int32),
                ("max_visits", C.c_int32), ("device", C.c_int32), ("seed", C.c_uint64),
                ("game_id_base", C.c_uint32), ("nn_mode", C.c_int32), ("sample_capacity_games", C.c_int32),
                ("reserved", C.c_int32 * 3)]


class GameInfo(C.Structure):
    _fields_ = [(n, C.c_int32) for n in
                ("A", "VS", "FS", "ML", "max_plies", "pos_image_bytes", "rec_bytes", "reserved")]


class SelfplayStats(C.Structure):
    _fields_ = [("nsamples", C.c_int64), ("total_plies", C.c_int64), ("wins", C.c_int64), ("draws", C.c_int64),
                ("losses", C.c_int64), ("rollouts", C.c_int64), ("plies", C.c_int32), ("faults", C.c_int32),
                ("search_seconds", C.c_double), ("total_seconds", C.c_double)]


class LogProbArgs(C.Structure):                     # agz_logprob_args
    _fields_ = [("n", C.c_int64), ("a", C.c_int64), ("logits", C.c_void_p), ("ld", C.c_int64), ("dtype", C.c_int32), ("top", C.c_int32),
                ("mask", C.c_void_p), ("ld_mask", C.c_int64), ("moves", C.c_void_p), ("target", C.c_void_p), ("ld_target", C.c_int64),
                ("move_logp", C.c_void_p), ("entropy", C.c_void_p), ("target_logp", C.c_void_p), ("top_logp", C.c_void_p),
                ("top_move", C.c_void_p), ("stats", C.c_void_p), ("workspace", C.c_void_p), ("workspace_bytes", C.c_int64)]


class LinearFp8Args(C.Structure):                   # agz_linear_fp8_args
    _fields_ = [("m", C.c_int64), ("n", C.c_int64), ("k", C.c_int64), ("x", C.c_void_p), ("ldx", C.c_int64), ("w", C.c_void_p), ("ldw", C.c_int64),
                ("bias", C.c_void_p), ("dtype", C.c_int32), ("w_dtype", C.c_int32), ("bias_dtype", C.c_int32), ("relu", C.c_int32)]


class AdamWOptions(C.Structure):                    # agz_adamw_options
    _fields_ = [("lr", C.c_double), ("beta1", C.c_double), ("beta2", C.c_double), ("eps", C.c_double), ("weight_decay", C.c_double),
                ("param_dtype", C.c_int32), ("grad_dtype", C.c_int32), ("bits", C.c_int32), ("seed", C.c_uint32), ("tensor_base", C.c_int32),
                ("step", C.c_int64), ("step_dev", C.c_void_p)]


def build_library():
    """Compile libagz.so for gfx950 (hipcc cross-compiles without a GPU)."""
    subprocess.check_call(["make", "-s", "-C", CSRC])


def load_library():
    global _LIB
    if _LIB is not None:
        return _LIB
    if not os.path.exists(LIB_PATH):
        raise LibraryMissing(f"{LIB_PATH} not found: build it with `make -C {CSRC}` "
                             "(alphagpu_amd has no CPU fallback)")
    L = C.CDLL(LIB_PATH)
    vp, f32p = C.c_void_p, C.c_void_p
    L.agz_query_game.argtypes = [C.POINTER(Config), C.POINTER(GameInfo)]
    L.agz_create.argtypes = [C.POINTER(Config), C.POINTER(vp)]
    L.agz_destroy.argtypes = [vp]
    L.agz_destroy.restype = None
    L.agz_last_error.argtypes = [vp]
    L.agz_last_error.restype = C.c_char_p
    L.agz_get_info.argtypes = [vp, C.POINTER(GameInfo)]
    L.agz_set_network.argtypes = [vp, C.c_int, C.c_int] + [f32p] * 6
    L.agz_set_network_slot.argtypes = [vp, C.c_int, C.c_int, C.c_int] + [f32p] * 6
    L.agz_init_weights.argtypes = [C.c_uint64, C.c_int, C.c_int, C.c_int, C.c_int] + [f32p] * 6
    L.agz_set_roots.argtypes = [vp, vp, C.c_int, vp, C.c_int]
    L.agz_search.argtypes = [vp, C.c_int, C.c_float, C.c_int, C.c_uint32]
    L.agz_search_actor.argtypes = [vp, C.c_int, C.c_int, C.c_float, C.c_int, C.c_uint32]
    L.agz_search_begin.argtypes = [vp, C.c_float, C.c_int, C.c_uint32]
    L.agz_rollout_select.argtypes = [vp, C.c_uint32, C.c_int]
    L.agz_rollout_eval.argtypes = [vp]
    L.agz_get_eval.argtypes = [vp, f32p, f32p]
    L.agz_inject_eval.argtypes = [vp, f32p, f32p]
    L.agz_get_logits.argtypes = [vp, f32p, f32p]
    L.agz_set_seed.argtypes = [vp, C.c_uint64]
    L.agz_get_search_form.argtypes = [vp, C.c_char_p, C.c_char_p, C.c_int]
    L.agz_rollout_expand_backup.argtypes = [vp]
    L.agz_search_end.argtypes = [vp]
    for n in ("policy", "batch", "leaf_batch", "root_visits", "root_q", "leaf", "node_count"):
        getattr(L, "agz_get_" + n).argtypes = [vp, vp]
    L.agz_get_counters.argtypes = [vp, C.POINTER(C.c_uint64), C.POINTER(C.c_uint64), C.POINTER(C.c_uint64)]
    L.agz_selfplay.argtypes = [vp, C.c_int, C.c_int, C.c_float, C.c_int, C.POINTER(SelfplayStats)]
    L.agz_selfplay_chain.argtypes = [vp, C.c_int, C.c_int, C.c_int, C.c_float, C.c_int, C.POINTER(SelfplayStats)]
    L.agz_duel.argtypes = [vp, C.c_int, C.c_int, C.c_float, C.c_int, C.c_int, C.POINTER(C.c_int64 * 3)]
    L.agz_get_samples.argtypes = [vp] + [vp] * 8
    L.agz_get_samples_packed.argtypes = [vp, vp, C.c_int64, C.POINTER(C.c_int64)]
    L.agz_unpack_records.argtypes = [C.POINTER(GameInfo), vp, C.c_int64] + [vp] * 8
    L.agz_perft.argtypes = [C.POINTER(Config), C.c_int, C.POINTER(C.c_int64), C.POINTER(C.c_int64 * 3)]
    L.agz_stream.argtypes = [vp]
    L.agz_stream.restype = vp
    L.agz_synchronize.argtypes = [vp]
    L.agz_get_kernel_times.argtypes = [vp, C.POINTER(C.c_double), C.POINTER(C.c_double), C.POINTER(C.c_int64), C.c_int]
    L.agz_set_profiling.argtypes = [vp, C.c_int]
    L.agz_get_tree_busy_ms.argtypes = [vp, C.POINTER(C.c_double)]
    L.agz_get_nn_leaves.argtypes = [vp, C.POINTER(C.c_uint64)]
    L.agz_set_network_tag.argtypes = [vp, C.c_uint32]
    i64p = C.POINTER(C.c_int64)
    L.agz_comm_unique_id.argtypes = [vp]
    L.agz_comm_create.argtypes = [vp, C.c_int, C.c_int, vp, C.c_int64, C.POINTER(vp)]
    L.agz_comm_destroy.argtypes = [vp]
    L.agz_comm_destroy.restype = None
    L.agz_comm_last_error.argtypes = [vp]
    L.agz_comm_last_error.restype = C.c_char_p
    L.agz_allgather_samples.argtypes = [vp, vp, i64p]
    L.agz_allgather_samples_start.argtypes = [vp, vp, C.c_int64]
    L.agz_allgather_samples_wait.argtypes = [vp, i64p, i64p]
    L.agz_comm_fetch_records.argtypes = [vp, C.c_int, vp, C.c_int64, C.c_int64]
    L.agz_comm_records_device.argtypes = [vp, C.c_int]
    L.agz_comm_records_device.restype = vp
    L.agz_get_age_stats.argtypes = [vp, C.POINTER(C.c_uint64 * 3)]
    if hasattr(L, "agz_comm_post_status") or not os.environ.get("AGZ_LIB_PATH"):   # (an A/B library named by AGZ_LIB_PATH may be a build of an earlier round)
        L.agz_get_samples_packed_async.argtypes = [vp, vp, C.c_int64, C.POINTER(C.c_int64)]
        L.agz_comm_post_status.argtypes = [vp, C.c_int]
        L.agz_comm_get_statuses.argtypes = [vp, C.POINTER(C.c_int32)]
        L.agz_allgather_samples_status.argtypes = [vp, vp, C.c_int, i64p, C.POINTER(C.c_int32)]
    if hasattr(L, "agz_adamw_step_missed") or not os.environ.get("AGZ_LIB_PATH"):
        i64, i32 = C.c_int64, C.c_int
        L.agz_ops_last_error.argtypes = []
        L.agz_ops_last_error.restype = C.c_char_p
        L.agz_logprob_workspace.argtypes = [i64, i64, C.c_int32]
        L.agz_logprob_forward.argtypes = [i32, vp, vp]
        L.agz_logprob_backward.argtypes = [i32, vp, vp, vp, vp, vp, vp, vp, i64]
        L.agz_fp8_pitch.argtypes = L.agz_fp8_scale_pitch.argtypes = [i64]
        L.agz_fp8_colsum_ws.argtypes = [i64, i64]
        L.agz_fp8_quantize.argtypes = [i32, vp, vp, i32, i64, i64, i64, vp, i32, vp, vp, vp, vp, vp, vp, i64]
        L.agz_fp8_matmul_workspace.argtypes = [i64, i64, i64]
        L.agz_fp8_matmul.argtypes = [i32, vp, i64, i64, i64, vp, vp, vp, vp, vp, i32, i32, vp, i32, i64, vp, i64]
        L.agz_linear_fp8_workspace.argtypes = [i64] * 3
        L.agz_linear_fp8_saved.argtypes = [i64] * 3 + [i32] * 2
        L.agz_linear_fp8_backward_workspace.argtypes = [i64] * 3 + [i32] * 3
        L.agz_linear_fp8_apply_workspace.argtypes = [i64] * 3
        L.agz_linear_fp8_apply.argtypes = [i32, vp, vp, vp, vp, vp, vp, i64]
        L.agz_linear_fp8_forward.argtypes = [i32, vp, vp, vp, vp, i32, i32, vp, i64]
        L.agz_linear_fp8_backward.argtypes = [i32, vp, vp, vp, vp, vp, i32, i32, vp, vp, vp, vp, i64]
        L.agz_adamw_state_elements.argtypes = [i32, vp]
        L.agz_adamw_step.argtypes = [i32, vp, vp, i32, vp, vp, vp, vp, vp, vp, vp]
        L.agz_adamw_step_missed.argtypes = [i32, vp, vp, vp, vp, i32, vp, vp, vp, vp, vp, vp, vp]
        for n in ("logprob_workspace", "fp8_pitch", "fp8_scale_pitch", "fp8_colsum_ws", "fp8_matmul_workspace", "linear_fp8_workspace", "linear_fp8_saved", "linear_fp8_apply_workspace", "linear_fp8_backward_workspace", "adamw_state_elements"):
            getattr(L, "agz_" + n).restype = i64
    _LIB = L
    return L
