"""ctypes view of the C ABI in include/hogwild_hip.h.

The library is required: importing this module without a built libhogwild_hip.so raises, and no entry
point here has a CPU or eager fallback.  Tensors are torch tensors on the GPU; only their pointers,
sizes and the current HIP stream cross the boundary.
"""
from __future__ import annotations

import ctypes as C
import os
from typing import List, Optional, Sequence

import torch

_HERE = os.path.dirname(os.path.abspath(__file__))
LIB_PATH = os.path.join(_HERE, "libhogwild_hip.so")

HW_MAX_FRAGMENTS = 512          # per call
HW_MAX_LAUNCH_FRAGMENTS = 64    # per attention launch (what hw_plan describes)
HW_ABI_VERSION = 6              # the version the structures below mirror
HW_MAX_SPLITS = 256
HW_STATIC_SCRATCH_BYTES = 8 << 20
HW_F32, HW_F16, HW_BF16 = 0, 1, 2
_DTYPE_CODE = {torch.float32: HW_F32, torch.float16: HW_F16, torch.bfloat16: HW_BF16}

EXPORTS = [
    "hw_version", "hw_status_string", "hw_validate", "hw_plan_debug", "hw_workspace_bytes",
    "hw_fused_attention", "hw_fused_attention_stages", "hw_sdpa", "hw_rope", "hw_device_cus",
    "hw_paged_validate", "hw_paged_plan_debug", "hw_paged_workspace_bytes", "hw_paged_sdpa", "hw_varlen_paged_sdpa",
    "hw_paged_sdpa_stages", "hw_copy_to_blocks", "hw_build_inputs", "hw_rope_append",
    "hw_build_inputs_dev", "hw_advance_lengths", "hw_stream_capture_id", "hw_fused_attention_static", "hw_sdpa_workspace_bytes",
    "hw_merge_segments",
    "hw_copy_to_blocks_q4", "hw_read_blocks_q4", "hw_paged_q4_validate", "hw_paged_q4_plan_debug", "hw_paged_q4_workspace_bytes",
    "hw_paged_sdpa_q4", "hw_varlen_paged_sdpa_q4",
    "hw_window_validate", "hw_window_plan_debug", "hw_window_workspace_bytes", "hw_window_paged_sdpa", "hw_window_varlen_paged_sdpa",
    "hw_trim_blocks", "hw_packed_slots", "hw_copy_to_slots", "hw_verify_workspace_bytes", "hw_verify_drafts",
    "hw_pool_workspace_bytes", "hw_fork_blocks", "hw_free_blocks", "hw_reserve_blocks", "hw_reserve_step", "hw_compact_blocks", "hw_copy_pages",
]


class HwProblem(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32),
        ("F", C.c_int32), ("W", C.c_int32), ("Hq", C.c_int32), ("Hkv", C.c_int32), ("S", C.c_int32),
        ("E", C.c_int32), ("Ev", C.c_int32), ("RotE", C.c_int32),
        ("scale", C.c_float),
        ("out", C.c_void_p), ("lse", C.c_void_p), ("rq", C.c_void_p),
        ("q", C.c_void_p), ("locations", C.c_void_p), ("cosines", C.c_void_p), ("sines", C.c_void_p),
        ("k", C.POINTER(C.c_void_p)), ("v", C.POINTER(C.c_void_p)), ("len", C.POINTER(C.c_int32)),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("splits", C.c_int32), ("row_blocks", C.c_int32),
        ("cap", C.POINTER(C.c_int32)),
        ("len_dev", C.c_void_p),
        ("variant", C.c_int32),
    ]


class HwPlan(C.Structure):
    _fields_ = [
        ("rows", C.c_int32), ("row_blocks", C.c_int32), ("row_groups", C.c_int32), ("tile_tokens", C.c_int32),
        ("tiles_per_head", C.c_int32), ("wgs_per_head", C.c_int32), ("workgroups", C.c_int32),
        ("tile_begin", C.c_int32 * (HW_MAX_LAUNCH_FRAGMENTS + 1)),
        ("wg_tile_begin", C.c_int32 * (HW_MAX_SPLITS + 1)),
        ("workspace_bytes", C.c_size_t),
    ]


class HwPagedProblem(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32),
        ("F", C.c_int32), ("W", C.c_int32), ("Hq", C.c_int32), ("Hkv", C.c_int32), ("E", C.c_int32), ("Ev", C.c_int32),
        ("S", C.c_int32), ("total_q", C.c_int32),
        ("block_size", C.c_int32), ("max_blocks", C.c_int32), ("num_blocks", C.c_int32),
        ("scale", C.c_float),
        ("out", C.c_void_p), ("lse", C.c_void_p), ("q", C.c_void_p), ("locations", C.c_void_p),
        ("fragment_lengths", C.c_void_p), ("key_cache", C.c_void_p), ("value_cache", C.c_void_p),
        ("block_table", C.c_void_p), ("cu_seqlens_q", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("splits", C.c_int32), ("row_blocks", C.c_int32),
    ]


class HwPagedPlan(C.Structure):
    _fields_ = [
        ("rows", C.c_int32), ("row_blocks", C.c_int32), ("row_groups", C.c_int32), ("splits", C.c_int32),
        ("workgroups", C.c_int32), ("device_planned", C.c_int32), ("workspace_bytes", C.c_size_t),
    ]


class HwCopyBlocks(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32),
        ("B", C.c_int32), ("Hkv", C.c_int32), ("S_new", C.c_int32), ("E", C.c_int32), ("Ev", C.c_int32),
        ("block_size", C.c_int32), ("max_blocks", C.c_int32), ("num_blocks", C.c_int32),
        ("key_states", C.c_void_p), ("value_states", C.c_void_p),
        ("ks_b", C.c_int64), ("ks_h", C.c_int64), ("ks_s", C.c_int64),
        ("vs_b", C.c_int64), ("vs_h", C.c_int64), ("vs_s", C.c_int64),
        ("key_cache", C.c_void_p), ("value_cache", C.c_void_p),
        ("block_table", C.c_void_p), ("seq_lengths", C.c_void_p),
    ]


class HwWindowProblem(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32),
        ("W", C.c_int32), ("Hq", C.c_int32), ("Hkv", C.c_int32), ("D", C.c_int32), ("S", C.c_int32), ("total_q", C.c_int32),
        ("block_size", C.c_int32), ("max_blocks", C.c_int32), ("num_blocks", C.c_int32),
        ("window", C.c_int32), ("sinks", C.c_int32),
        ("scale", C.c_float),
        ("out", C.c_void_p), ("lse", C.c_void_p), ("q", C.c_void_p), ("locations", C.c_void_p),
        ("key_cache", C.c_void_p), ("value_cache", C.c_void_p), ("block_table", C.c_void_p), ("cu_seqlens_q", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("splits", C.c_int32), ("row_blocks", C.c_int32),
    ]


class HwPackedBatch(C.Structure):
    _fields_ = [
        ("W", C.c_int32), ("max_blocks", C.c_int32), ("num_blocks", C.c_int32), ("block_size", C.c_int32), ("total", C.c_int32),
        ("block_table", C.c_void_p), ("positions", C.c_void_p), ("n_new", C.c_void_p),
        ("cu_seqlens", C.c_void_p), ("locations", C.c_void_p), ("slots", C.c_void_p),
    ]


class HwCopySlots(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32),
        ("total", C.c_int32), ("Hkv", C.c_int32), ("E", C.c_int32), ("Ev", C.c_int32), ("block_size", C.c_int32), ("num_blocks", C.c_int32),
        ("key_states", C.c_void_p), ("value_states", C.c_void_p),
        ("ks_t", C.c_int64), ("ks_h", C.c_int64), ("vs_t", C.c_int64), ("vs_h", C.c_int64),
        ("key_cache", C.c_void_p), ("value_cache", C.c_void_p), ("slots", C.c_void_p),
    ]


class HwVerify(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32), ("token_bytes", C.c_int32),
        ("W", C.c_int32), ("K", C.c_int32), ("V", C.c_int32),
        ("drafts", C.c_void_p), ("target", C.c_void_p), ("draft_probs", C.c_void_p),
        ("tp_w", C.c_int64), ("tp_k", C.c_int64), ("dp_w", C.c_int64), ("dp_k", C.c_int64),
        ("uniforms", C.c_void_p), ("n_drafts", C.c_void_p), ("positions", C.c_void_p), ("seq_lengths", C.c_void_p),
        ("tokens", C.c_void_p), ("accepted", C.c_void_p),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
        ("n_new", C.c_void_p),
    ]


class HwPool(C.Structure):
    _fields_ = [
        ("W", C.c_int32), ("max_blocks", C.c_int32), ("num_blocks", C.c_int32), ("block_size", C.c_int32),
        ("block_table", C.c_void_p), ("seq_lengths", C.c_void_p), ("ref_counts", C.c_void_p),
        ("caches", C.POINTER(C.c_void_p)), ("page_bytes", C.POINTER(C.c_size_t)), ("n_caches", C.c_int32),
        ("workspace", C.c_void_p), ("workspace_bytes", C.c_size_t),
    ]


class HwAppend(C.Structure):
    _fields_ = [
        ("dtype", C.c_int32), ("cs_dtype", C.c_int32), ("mode", C.c_int32),
        ("W", C.c_int32), ("Hkv", C.c_int32), ("S", C.c_int32), ("E", C.c_int32), ("Ev", C.c_int32), ("RotE", C.c_int32),
        ("key_states", C.c_void_p), ("value_states", C.c_void_p),
        ("ks_w", C.c_int64), ("ks_h", C.c_int64), ("ks_s", C.c_int64),
        ("vs_w", C.c_int64), ("vs_h", C.c_int64), ("vs_s", C.c_int64),
        ("cosines", C.c_void_p), ("sines", C.c_void_p),
        ("cs_w", C.c_int64), ("cs_s", C.c_int64),
        ("k_dst", C.POINTER(C.c_void_p)), ("v_dst", C.POINTER(C.c_void_p)),
        ("dst_len", C.POINTER(C.c_int32)), ("dst_cap", C.POINTER(C.c_int32)), ("n_new", C.POINTER(C.c_int32)),
        ("len_dev", C.c_void_p),
    ]


HW_ROPE_EAGER, HW_ROPE_FUSED = 0, 1
HW_VARIANT_MFMA, HW_VARIANT_VALU_QK = 0, 1


class HogwildError(RuntimeError):
    def __init__(self, status: int, where: str):
        self.status = status
        super().__init__(f"{where}: status {status}: {status_string(status)}")


def _load() -> C.CDLL:
    if not os.path.exists(LIB_PATH):
        raise ImportError(
            f"{LIB_PATH} is missing: build it with `python -m inference_lib_amd.build` "
            "(there is no fallback path for the Hogwild attention operators)")
    lib = C.CDLL(LIB_PATH)
    lib.hw_version.restype = C.c_int
    if lib.hw_version() != HW_ABI_VERSION:      # a stale library would be driven with structures of another layout
        raise ImportError(f"{LIB_PATH} has ABI version {lib.hw_version()}, this module mirrors version {HW_ABI_VERSION}: "
                          "rebuild it with `python -m inference_lib_amd.build`")
    lib.hw_status_string.restype = C.c_char_p
    lib.hw_status_string.argtypes = [C.c_int]
    lib.hw_validate.argtypes = [C.POINTER(HwProblem), C.c_int]
    lib.hw_plan_debug.argtypes = [C.POINTER(HwProblem), C.c_int, C.POINTER(HwPlan)]
    lib.hw_workspace_bytes.argtypes = [C.POINTER(HwProblem), C.POINTER(C.c_size_t)]
    lib.hw_sdpa_workspace_bytes.argtypes = [C.POINTER(HwProblem), C.POINTER(C.c_size_t)]
    lib.hw_fused_attention.argtypes = [C.POINTER(HwProblem), C.c_void_p]
    lib.hw_sdpa.argtypes = [C.POINTER(HwProblem), C.c_void_p]
    lib.hw_fused_attention_static.argtypes = [C.POINTER(HwProblem), C.c_void_p]
    lib.hw_fused_attention_stages.argtypes = [C.POINTER(HwProblem), C.c_void_p, C.c_int]
    lib.hw_rope.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.c_int, C.c_int, C.c_int, C.c_int,
                            C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.hw_paged_validate.argtypes = [C.POINTER(HwPagedProblem)]
    lib.hw_paged_plan_debug.argtypes = [C.POINTER(HwPagedProblem), C.c_int, C.POINTER(HwPagedPlan)]
    lib.hw_paged_workspace_bytes.argtypes = [C.POINTER(HwPagedProblem), C.POINTER(C.c_size_t)]
    lib.hw_paged_sdpa.argtypes = [C.POINTER(HwPagedProblem), C.c_void_p]
    lib.hw_varlen_paged_sdpa.argtypes = [C.POINTER(HwPagedProblem), C.c_void_p]
    lib.hw_paged_sdpa_stages.argtypes = [C.POINTER(HwPagedProblem), C.c_void_p, C.c_int]
    lib.hw_copy_to_blocks.argtypes = [C.POINTER(HwCopyBlocks), C.c_void_p]
    lib.hw_build_inputs.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.POINTER(C.c_int32), C.c_void_p, C.c_float, C.c_int,
                                    C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.hw_rope_append.argtypes = [C.POINTER(HwAppend), C.c_void_p]
    lib.hw_build_inputs_dev.argtypes = [C.c_void_p, C.c_void_p, C.c_void_p, C.c_void_p, C.POINTER(C.c_int32), C.c_void_p, C.c_float,
                                        C.c_int, C.c_int, C.c_int, C.c_int, C.c_int, C.c_void_p]
    lib.hw_advance_lengths.argtypes = [C.c_void_p, C.POINTER(C.c_int32), C.c_int, C.c_void_p]
    lib.hw_stream_capture_id.argtypes = [C.c_void_p, C.POINTER(C.c_ulonglong)]
    lib.hw_copy_to_blocks_q4.argtypes = [C.POINTER(HwCopyBlocks), C.c_void_p]
    lib.hw_read_blocks_q4.argtypes = [C.POINTER(HwCopyBlocks), C.c_void_p]
    lib.hw_paged_q4_validate.argtypes = [C.POINTER(HwPagedProblem)]
    lib.hw_paged_q4_plan_debug.argtypes = [C.POINTER(HwPagedProblem), C.c_int, C.POINTER(HwPagedPlan)]
    lib.hw_paged_q4_workspace_bytes.argtypes = [C.POINTER(HwPagedProblem), C.POINTER(C.c_size_t)]
    lib.hw_paged_sdpa_q4.argtypes = [C.POINTER(HwPagedProblem), C.c_void_p]
    lib.hw_varlen_paged_sdpa_q4.argtypes = [C.POINTER(HwPagedProblem), C.c_void_p]
    lib.hw_window_validate.argtypes = [C.POINTER(HwWindowProblem)]
    lib.hw_window_plan_debug.argtypes = [C.POINTER(HwWindowProblem), C.c_int, C.POINTER(HwPagedPlan)]
    lib.hw_window_workspace_bytes.argtypes = [C.POINTER(HwWindowProblem), C.POINTER(C.c_size_t)]
    lib.hw_window_paged_sdpa.argtypes = [C.POINTER(HwWindowProblem), C.c_void_p]
    lib.hw_window_varlen_paged_sdpa.argtypes = [C.POINTER(HwWindowProblem), C.c_void_p]
    lib.hw_trim_blocks.argtypes = [C.POINTER(HwPool), C.c_int, C.c_int, C.c_void_p]
    lib.hw_packed_slots.argtypes = [C.POINTER(HwPackedBatch), C.c_void_p]
    lib.hw_copy_to_slots.argtypes = [C.POINTER(HwCopySlots), C.c_void_p]
    lib.hw_verify_workspace_bytes.argtypes = [C.POINTER(HwVerify), C.POINTER(C.c_size_t)]
    lib.hw_verify_drafts.argtypes = [C.POINTER(HwVerify), C.c_void_p]
    lib.hw_pool_workspace_bytes.argtypes = [C.POINTER(HwPool), C.POINTER(C.c_size_t)]
    lib.hw_fork_blocks.argtypes = [C.POINTER(HwPool), C.c_void_p, C.c_void_p]
    lib.hw_free_blocks.argtypes = [C.POINTER(HwPool), C.c_void_p, C.c_void_p]
    lib.hw_reserve_blocks.argtypes = [C.POINTER(HwPool), C.c_void_p, C.c_void_p, C.c_void_p]
    lib.hw_reserve_step.argtypes = [C.POINTER(HwPool), C.c_void_p, C.c_int32, C.c_void_p, C.c_void_p, C.c_void_p]
    lib.hw_compact_blocks.argtypes = [C.POINTER(HwPool), C.c_void_p, C.c_void_p]
    lib.hw_copy_pages.argtypes = [C.POINTER(C.c_void_p), C.POINTER(C.c_size_t), C.c_int, C.c_int, C.POINTER(C.c_int32), C.POINTER(C.c_int32), C.c_int, C.c_void_p]
    return lib


lib = _load()


def status_string(status: int) -> str:
    return lib.hw_status_string(int(status)).decode()


def check(status: int, where: str) -> None:
    if status != 0:
        raise HogwildError(status, where)


def fragment_capacity(k: torch.Tensor, v: torch.Tensor) -> Optional[int]:
    """Row capacity of a fragment whose tensors [Hkv, L, D] are views into [Hkv, cap, D] allocations (rows contiguous,
    kv heads `cap` rows apart), or None if the pair is not of that form.  Packed fragments give cap == L."""
    Hkv, L, E = k.shape
    Ev = v.size(2)
    if L == 0:
        return 0
    if (E > 1 and k.stride(2) != 1) or (Ev > 1 and v.stride(2) != 1) or (L > 1 and (k.stride(1) != E or v.stride(1) != Ev)):
        return None
    if Hkv == 1:
        return L
    if k.stride(0) % E != 0 or v.stride(0) % Ev != 0 or k.stride(0) // E != v.stride(0) // Ev or k.stride(0) // E < L:
        return None
    return k.stride(0) // E


def _frag3(t: torch.Tensor) -> torch.Tensor:
    """Fragments come as [Hkv, L, D] or [1, Hkv, L, D] (src/binding.cu:85-94)."""
    if t.dim() == 4:
        if t.size(0) != 1:
            raise ValueError("4-D KV fragment must have a leading dimension of 1")
        return t[0]
    if t.dim() != 3:
        raise ValueError("KV fragment must be [Hkv, L, D] or [1, Hkv, L, D]")
    return t


class Problem:
    """Owns the ctypes arrays of one hw_problem and keeps the tensors alive."""

    def __init__(self, *, q: torch.Tensor, locations: torch.Tensor, keys: Sequence[torch.Tensor],
                 values: Sequence[torch.Tensor], scale: float, out: torch.Tensor,
                 cosines: Optional[torch.Tensor] = None, sines: Optional[torch.Tensor] = None,
                 rq: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 prerotated: bool = False, splits: int = 0, row_blocks: int = 0, len_dev: Optional[torch.Tensor] = None,
                 variant: int = 0):
        keys = [_frag3(k) for k in keys]
        values = [_frag3(v) for v in values]
        F = len(keys)
        if len(values) != F or locations.size(0) != F:
            raise ValueError("fragment count mismatch between keys, values and locations")
        if F < 1 or F > HW_MAX_FRAGMENTS:
            raise HogwildError(-5, "Problem")
        W, Hq, S, Ev = out.shape
        E = q.size(-1)
        Hkv = keys[0].size(0)
        if out.dtype not in _DTYPE_CODE:
            raise HogwildError(-2, "Problem")
        expect_q = (F, W, Hq, S, E) if prerotated else (W, Hq, S, E)
        if tuple(q.shape) != expect_q:
            raise ValueError(f"queries have shape {tuple(q.shape)}, expected {expect_q}")
        if tuple(locations.shape) != (F, W, S) or locations.dtype != torch.int32:
            raise ValueError("locations must be int32 [F, W, S]")
        tensors = [out, q, locations]
        caps = []
        for f in range(F):
            if keys[f].size(0) != Hkv or values[f].size(0) != Hkv or keys[f].size(1) != values[f].size(1) \
                    or keys[f].size(2) != E or values[f].size(2) != Ev:
                raise ValueError(f"fragment {f} has inconsistent shape")
            if keys[f].dtype != out.dtype or values[f].dtype != out.dtype:
                raise ValueError("KV fragments must have the dtype of the output")
            cap = fragment_capacity(keys[f], values[f])
            if cap is None:
                raise ValueError(f"fragment {f}: rows must be contiguous and kv heads a whole number of rows apart "
                                 "(the same number for keys and values)")
            caps.append(cap)
            if keys[f].device != out.device or values[f].device != out.device:
                raise ValueError("all tensors must live on the output's device")
        if q.dtype != out.dtype:
            raise ValueError("queries must have the dtype of the output")
        rot = 0
        if not prerotated:
            if cosines is None or sines is None:
                raise ValueError("the fused operator needs cosines and sines")
            rot = cosines.size(-1)
            if tuple(cosines.shape) != (F, W, S, rot) or tuple(sines.shape) != (F, W, S, rot):
                raise ValueError("cosines / sines must be [F, W, S, RotE]")
            if cosines.dtype != torch.float32 or sines.dtype != torch.float32:
                raise ValueError("cosines / sines must be float32")
            tensors += [cosines, sines]
        if rq is not None:
            if tuple(rq.shape) != (F, W, Hq, S, E) or rq.dtype != out.dtype:
                raise ValueError("rotated-query buffer must be [F, W, Hq, S, E] in the output dtype")
            tensors.append(rq)
        if lse is not None:
            if tuple(lse.shape) != (W, Hq, S) or lse.dtype != torch.float32:
                raise ValueError("lse must be float32 [W, Hq, S]")
            tensors.append(lse)
        if len_dev is not None:      # current lengths in device memory; the fragment tensors then give the planned bounds
            if len_dev.dtype != torch.int32 or tuple(len_dev.shape) != (F,):
                raise ValueError("len_dev must be int32 [F]")
            tensors.append(len_dev)
        for t in tensors:
            if not t.is_contiguous():
                raise ValueError("all tensors must be contiguous")
            if t.device != out.device:
                raise ValueError("all tensors must live on the output's device")
        self._keep = tensors + keys + values
        self.device = out.device
        self._cap = (C.c_int32 * F)(*caps)
        self._k = (C.c_void_p * F)(*[k.data_ptr() for k in keys])
        self._v = (C.c_void_p * F)(*[v.data_ptr() for v in values])
        self._len = (C.c_int32 * F)(*[k.size(1) for k in keys])
        p = HwProblem()
        p.dtype = _DTYPE_CODE[out.dtype]
        p.F, p.W, p.Hq, p.Hkv, p.S, p.E, p.Ev, p.RotE = F, W, Hq, Hkv, S, E, Ev, rot
        p.scale = float(scale)
        p.out = out.data_ptr()
        p.lse = lse.data_ptr() if lse is not None else None
        p.rq = rq.data_ptr() if rq is not None else None
        p.q = q.data_ptr()
        p.locations = locations.data_ptr()
        p.cosines = cosines.data_ptr() if cosines is not None else None
        p.sines = sines.data_ptr() if sines is not None else None
        p.k = C.cast(self._k, C.POINTER(C.c_void_p))
        p.v = C.cast(self._v, C.POINTER(C.c_void_p))
        p.len = C.cast(self._len, C.POINTER(C.c_int32))
        p.cap = C.cast(self._cap, C.POINTER(C.c_int32))
        p.len_dev = len_dev.data_ptr() if len_dev is not None else None
        p.splits = int(splits)
        p.row_blocks = int(row_blocks)
        p.variant = int(variant)      # 0 = matrix cores; 1 = logits by VALU dot products (HW_VARIANT_VALU_QK, for A/B measurements)
        self.p = p
        self.prerotated = prerotated
        self._ws = None

    def workspace_bytes(self) -> int:
        n = C.c_size_t(0)
        with torch.cuda.device(self.device):
            fn = lib.hw_sdpa_workspace_bytes if self.prerotated else lib.hw_workspace_bytes
            check(fn(C.byref(self.p), C.byref(n)), fn.__name__)
        return n.value

    def set_workspace(self, ws: Optional[torch.Tensor] = None) -> None:
        if ws is None:
            ws = torch.empty(self.workspace_bytes(), dtype=torch.uint8, device=self.device)
        self._ws = ws
        self.p.workspace = ws.data_ptr()
        self.p.workspace_bytes = ws.numel() * ws.element_size()

    def run(self, stages: int = 3) -> None:
        """stages: 1 = attention kernel only (partials stay in the workspace), 2 = merge only, 3 = both."""
        if self._ws is None:
            self.set_workspace()
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream(self.device).cuda_stream
            if stages != 3:
                if self.prerotated:
                    raise ValueError("separate stages exist for the fused entry only")
                check(lib.hw_fused_attention_stages(C.byref(self.p), C.c_void_p(stream), stages), "hw_fused_attention_stages")
                return
            fn = lib.hw_sdpa if self.prerotated else lib.hw_fused_attention
            check(fn(C.byref(self.p), C.c_void_p(stream)), fn.__name__)


    def run_static(self) -> None:
        """hw_fused_attention_static: the same step with the partials in the library's own device array; allocates nothing."""
        if self.prerotated:
            raise ValueError("the static-scratch entry exists for the fused operator only")
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream(self.device).cuda_stream
            check(lib.hw_fused_attention_static(C.byref(self.p), C.c_void_p(stream)), "hw_fused_attention_static")


def plan(lens: Sequence[int], *, W: int, S: int, Hq: int, Hkv: int, Ev: int, num_cus: int, splits: int = 0,
         dtype: int = HW_BF16, row_blocks: int = 0) -> HwPlan:
    """Host-only split plan (no GPU needed)."""
    F = len(lens)
    arr = (C.c_int32 * max(F, 1))(*lens)
    p = HwProblem()
    p.F, p.W, p.S, p.Hq, p.Hkv, p.Ev, p.E = F, W, S, Hq, Hkv, Ev, Ev
    p.len = C.cast(arr, C.POINTER(C.c_int32))
    p.splits = splits
    p.dtype = dtype
    p.row_blocks = row_blocks
    out = HwPlan()
    check(lib.hw_plan_debug(C.byref(p), num_cus, C.byref(out)), "hw_plan_debug")
    return out


def q4_row_bytes(head_dim: int) -> int:
    """Bytes of one token's codes, scales and offsets in a 4-bit cache (HW_Q4_ROW_BYTES)."""
    return head_dim // 16 * 9


def check_q4_caches(key_cache: torch.Tensor, value_cache: torch.Tensor, head_dim: int) -> None:
    if key_cache.dtype != torch.uint8 or value_cache.dtype != torch.uint8:
        raise ValueError("4-bit caches must be uint8")
    if head_dim not in (64, 128, 256):
        raise HogwildError(-4, "4-bit caches")
    if key_cache.size(3) != q4_row_bytes(head_dim) or value_cache.size(3) != q4_row_bytes(head_dim):
        raise ValueError(f"4-bit caches of head dimension {head_dim} have rows of {q4_row_bytes(head_dim)} bytes")
    if key_cache.size(2) % 8 != 0:
        raise ValueError("the block size of a 4-bit cache must be a multiple of 8")


class PagedProblem:
    """One call of the paged attention operators (hw_paged_sdpa, or hw_varlen_paged_sdpa when cu_seqlens_q is given).

    fixed length:    q [F, W, Hq, S, E], locations [F, W, S], fragment_lengths [F], out [W, Hq, S, Ev], lse [W, Hq, S]
    variable length: q [F, T, Hq, E], locations [F, T], fragment_lengths [F, W], cu_seqlens_q [W+1], out [T, Hq, Ev],
                     lse [T, Hq]
    key_cache / value_cache [num_blocks, Hkv, block_size, E|Ev], block_table int32 [W, max_blocks]; with q4 = True uint8
    [num_blocks, Hkv, block_size, q4_row_bytes(E)] (hw_paged_sdpa_q4, hw_varlen_paged_sdpa_q4).
    """

    def __init__(self, *, q: torch.Tensor, locations: torch.Tensor, fragment_lengths: torch.Tensor,
                 key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor, scale: float,
                 out: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None, lse: Optional[torch.Tensor] = None,
                 splits: int = 0, row_blocks: int = 0, q4: bool = False):
        varlen = cu_seqlens_q is not None
        if out.dtype not in _DTYPE_CODE:
            raise HogwildError(-2, "PagedProblem")
        if key_cache.dim() != 4 or value_cache.dim() != 4 or key_cache.shape[:3] != value_cache.shape[:3]:
            raise ValueError("key_cache / value_cache must be [num_blocks, Hkv, block_size, E|Ev]")
        NB, Hkv, BS, E = key_cache.shape
        Ev = value_cache.size(3)
        if q4:
            E = Ev = q.size(-1)
            check_q4_caches(key_cache, value_cache, E)
        if block_table.dim() != 2:
            raise ValueError("block_table must be [W, max_blocks]")
        W = block_table.size(0)
        F = locations.size(0)
        if varlen:
            T, Hq = out.size(0), out.size(1)
            S = 0
            if tuple(out.shape) != (T, Hq, Ev) or tuple(q.shape) != (F, T, Hq, E) or tuple(locations.shape) != (F, T):
                raise ValueError("variable-length layout: q [F,T,Hq,E], locations [F,T], out [T,Hq,Ev]")
            if tuple(fragment_lengths.shape) != (F, W) or tuple(cu_seqlens_q.shape) != (W + 1,):
                raise ValueError("variable-length layout: fragment_lengths [F,W], cu_seqlens_q [W+1]")
            lse_shape = (T, Hq)
        else:
            if out.dim() != 4 or out.size(0) != W:
                raise ValueError("out must be [W, Hq, S, Ev] with one block-table row per worker")
            _, Hq, S, _ = out.shape
            T = 0
            if tuple(out.shape) != (W, Hq, S, Ev) or tuple(q.shape) != (F, W, Hq, S, E) or tuple(locations.shape) != (F, W, S):
                raise ValueError("fixed-length layout: q [F,W,Hq,S,E], locations [F,W,S], out [W,Hq,S,Ev]")
            if tuple(fragment_lengths.shape) != (F,):
                raise ValueError("fixed-length layout: fragment_lengths [F]")
            lse_shape = (W, Hq, S)
        tensors = [out, q, locations, fragment_lengths, key_cache, value_cache, block_table]
        if varlen:
            tensors.append(cu_seqlens_q)
        if lse is not None:
            if tuple(lse.shape) != lse_shape or lse.dtype != torch.float32:
                raise ValueError(f"lse must be float32 {lse_shape}")
            tensors.append(lse)
        for t in (locations, fragment_lengths, block_table) + ((cu_seqlens_q,) if varlen else ()):
            if t.dtype != torch.int32:
                raise ValueError("locations, fragment_lengths, block_table and cu_seqlens_q must be int32")
        for t in (q,) if q4 else (q, key_cache, value_cache):
            if t.dtype != out.dtype:
                raise ValueError("queries and caches must have the dtype of the output")
        for t in tensors:
            if not t.is_contiguous():
                raise ValueError("all tensors must be contiguous")
            if t.device != out.device:
                raise ValueError("all tensors must live on the output's device")
        self._keep = tensors
        self.device = out.device
        p = HwPagedProblem()
        p.dtype = _DTYPE_CODE[out.dtype]
        p.F, p.W, p.Hq, p.Hkv, p.E, p.Ev, p.S, p.total_q = F, W, Hq, Hkv, E, Ev, S, T
        p.block_size, p.max_blocks, p.num_blocks = BS, block_table.size(1), NB
        p.scale = float(scale)
        p.out = out.data_ptr()
        p.lse = lse.data_ptr() if lse is not None else None
        p.q = q.data_ptr()
        p.locations = locations.data_ptr()
        p.fragment_lengths = fragment_lengths.data_ptr()
        p.key_cache = key_cache.data_ptr()
        p.value_cache = value_cache.data_ptr()
        p.block_table = block_table.data_ptr()
        p.cu_seqlens_q = cu_seqlens_q.data_ptr() if varlen else None
        p.splits = int(splits)
        p.row_blocks = int(row_blocks)
        self.p = p
        self.varlen = varlen
        self.q4 = q4
        self._ws = None

    def workspace_bytes(self) -> int:
        n = C.c_size_t(0)
        with torch.cuda.device(self.device):
            if self.q4:
                check(lib.hw_paged_q4_validate(C.byref(self.p)), "hw_paged_q4_validate")
                check(lib.hw_paged_q4_workspace_bytes(C.byref(self.p), C.byref(n)), "hw_paged_q4_workspace_bytes")
            else:
                check(lib.hw_paged_workspace_bytes(C.byref(self.p), C.byref(n)), "hw_paged_workspace_bytes")
        return n.value

    def set_workspace(self, ws: Optional[torch.Tensor] = None) -> None:
        if ws is None:
            ws = torch.empty(max(self.workspace_bytes(), 256), dtype=torch.uint8, device=self.device)
        self._ws = ws
        self.p.workspace = ws.data_ptr()
        self.p.workspace_bytes = ws.numel() * ws.element_size()

    def run(self, stages: int = 3) -> None:
        if self._ws is None:
            self.set_workspace()
        with torch.cuda.device(self.device):
            stream = torch.cuda.current_stream(self.device).cuda_stream
            if stages != 3:
                if self.q4:
                    raise ValueError("separate stages exist for caches in 16 and 32 bits only")
                check(lib.hw_paged_sdpa_stages(C.byref(self.p), C.c_void_p(stream), stages), "hw_paged_sdpa_stages")
                return
            if self.q4:
                fn = lib.hw_varlen_paged_sdpa_q4 if self.varlen else lib.hw_paged_sdpa_q4
            else:
                fn = lib.hw_varlen_paged_sdpa if self.varlen else lib.hw_paged_sdpa
            check(fn(C.byref(self.p), C.c_void_p(stream)), fn.__name__)


def paged_plan(*, W: int, Hq: int, Hkv: int, Ev: int, block_size: int, max_blocks: int, num_cus: int, S: int = 0,
               total_q: Optional[int] = None, splits: int = 0, dtype: int = HW_BF16, row_blocks: int = 0, q4: bool = False) -> HwPagedPlan:
    """Host-only plan of the paged operators (no GPU needed); total_q selects the variable-length operator, q4 caches in 4 bits."""
    p = HwPagedProblem()
    p.dtype = dtype
    p.F, p.W, p.Hq, p.Hkv, p.E, p.Ev, p.S = 1, W, Hq, Hkv, Ev, Ev, S
    p.block_size, p.max_blocks, p.num_blocks = block_size, max_blocks, 1
    if total_q is not None:
        p.total_q = total_q
        p.cu_seqlens_q = 16       # only tested for being non-NULL by the planner
    p.splits = splits
    p.row_blocks = row_blocks
    out = HwPagedPlan()
    fn = lib.hw_paged_q4_plan_debug if q4 else lib.hw_paged_plan_debug
    check(fn(C.byref(p), num_cus, C.byref(out)), fn.__name__)
    return out


def copy_to_blocks(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                   block_table: torch.Tensor, seq_lengths: torch.Tensor, q4: bool = False) -> None:
    """Append key_states / value_states [B, Hkv, S_new, E|Ev] (any strides with a contiguous last dimension) to the
    paged caches at positions seq_lengths[b] + t; with q4 to caches in 4 bits."""
    if key_states.dim() != 4 or value_states.dim() != 4 or key_states.shape[:3] != value_states.shape[:3]:
        raise ValueError("key_states / value_states must be [B, Hkv, S_new, E|Ev]")
    B, Hkv, S_new, E = key_states.shape
    Ev = value_states.size(3)
    if key_cache.dim() != 4 or value_cache.dim() != 4 or key_cache.size(1) != Hkv or key_cache.shape[:3] != value_cache.shape[:3] \
            or (not q4 and (key_cache.size(3) != E or value_cache.size(3) != Ev)):
        raise ValueError("caches must be [num_blocks, Hkv, block_size, E|Ev]")
    if key_states.dtype not in _DTYPE_CODE:
        raise HogwildError(-2, "copy_to_blocks")
    if q4:
        if E != Ev:
            raise ValueError("4-bit caches have one head dimension for keys and values")
        check_q4_caches(key_cache, value_cache, E)
    for t in (value_states,) if q4 else (value_states, key_cache, value_cache):
        if t.dtype != key_states.dtype:
            raise ValueError("states and caches must share one dtype")
    if tuple(seq_lengths.shape) != (B,) or block_table.dim() != 2 or block_table.size(0) != B:
        raise ValueError("block_table must be [B, max_blocks], seq_lengths [B]")
    for t in (block_table, seq_lengths):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("block_table and seq_lengths must be contiguous int32")
    if not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("caches must be contiguous")
    if (E > 1 and key_states.stride(3) != 1) or (Ev > 1 and value_states.stride(3) != 1):
        key_states, value_states = key_states.contiguous(), value_states.contiguous()
    for t in (key_states, value_states, value_cache, block_table, seq_lengths):
        if t.device != key_cache.device:
            raise ValueError("all tensors must live on the caches' device")
    c = HwCopyBlocks()
    c.dtype = _DTYPE_CODE[key_states.dtype]
    c.B, c.Hkv, c.S_new, c.E, c.Ev = B, Hkv, S_new, E, Ev
    c.block_size, c.max_blocks, c.num_blocks = key_cache.size(2), block_table.size(1), key_cache.size(0)
    c.key_states, c.value_states = key_states.data_ptr(), value_states.data_ptr()
    c.ks_b, c.ks_h, c.ks_s = key_states.stride(0), key_states.stride(1), key_states.stride(2)
    c.vs_b, c.vs_h, c.vs_s = value_states.stride(0), value_states.stride(1), value_states.stride(2)
    c.key_cache, c.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    c.block_table, c.seq_lengths = block_table.data_ptr(), seq_lengths.data_ptr()
    with torch.cuda.device(key_cache.device):
        stream = torch.cuda.current_stream(key_cache.device).cuda_stream
        fn = lib.hw_copy_to_blocks_q4 if q4 else lib.hw_copy_to_blocks
        check(fn(C.byref(c), C.c_void_p(stream)), fn.__name__)


def read_blocks_q4(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor,
                   block_table: torch.Tensor, seq_lengths: torch.Tensor) -> None:
    """Write the values of a 4-bit cache at positions seq_lengths[b] + t into key_states / value_states [B, Hkv, n, D]."""
    if key_states.dim() != 4 or key_states.shape != value_states.shape or not key_states.is_contiguous() or not value_states.is_contiguous():
        raise ValueError("key_states / value_states must be contiguous [B, Hkv, n, D]")
    if key_states.dtype not in _DTYPE_CODE or value_states.dtype != key_states.dtype:
        raise HogwildError(-2, "read_blocks_q4")
    B, Hkv, n, D = key_states.shape
    if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or key_cache.size(1) != Hkv or not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("caches must be contiguous [num_blocks, Hkv, block_size, row bytes]")
    check_q4_caches(key_cache, value_cache, D)
    if tuple(seq_lengths.shape) != (B,) or block_table.dim() != 2 or block_table.size(0) != B:
        raise ValueError("block_table must be [B, max_blocks], seq_lengths [B]")
    for t in (block_table, seq_lengths):
        if t.dtype != torch.int32 or not t.is_contiguous():
            raise ValueError("block_table and seq_lengths must be contiguous int32")
    for t in (key_states, value_states, value_cache, block_table, seq_lengths):
        if t.device != key_cache.device:
            raise ValueError("all tensors must live on the caches' device")
    c = HwCopyBlocks()
    c.dtype = _DTYPE_CODE[key_states.dtype]
    c.B, c.Hkv, c.S_new, c.E, c.Ev = B, Hkv, n, D, D
    c.block_size, c.max_blocks, c.num_blocks = key_cache.size(2), block_table.size(1), key_cache.size(0)
    c.key_states, c.value_states = key_states.data_ptr(), value_states.data_ptr()
    c.key_cache, c.value_cache = key_cache.data_ptr(), value_cache.data_ptr()
    c.block_table, c.seq_lengths = block_table.data_ptr(), seq_lengths.data_ptr()
    with torch.cuda.device(key_cache.device):
        stream = torch.cuda.current_stream(key_cache.device).cuda_stream
        check(lib.hw_read_blocks_q4(C.byref(c), C.c_void_p(stream)), "hw_read_blocks_q4")


class WindowProblem:
    """hw_window_problem: out and q [W, Hq, S, D], locations [W, S], lse [W, Hq, S], or, with cu_seqlens_q [W + 1], packed: out and q
    [total_q, Hq, D], locations [total_q], lse [total_q, Hq]."""

    def __init__(self, *, q: torch.Tensor, locations: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, block_table: torch.Tensor,
                 scale: float, window: int, sinks: int, out: torch.Tensor, cu_seqlens_q: Optional[torch.Tensor] = None,
                 lse: Optional[torch.Tensor] = None, splits: int = 0, row_blocks: int = 0):
        varlen = cu_seqlens_q is not None
        if out.dtype not in _DTYPE_CODE:
            raise HogwildError(-2, "WindowProblem")
        if key_cache.dim() != 4 or key_cache.shape != value_cache.shape or block_table.dim() != 2:
            raise ValueError("caches must be [num_blocks, Hkv, block_size, D], block_table [W, max_blocks]")
        W = block_table.size(0)
        if out.dim() != (3 if varlen else 4) or q.shape != out.shape or out.size(-1) != key_cache.size(3):
            raise ValueError("queries and output must be [W, Hq, S, D], or [total_q, Hq, D] with cu_seqlens_q")
        if not varlen and out.size(0) != W:
            raise ValueError("output must be [W, Hq, S, D] with one block-table row per sequence")
        if tuple(locations.shape) != ((out.size(0),) if varlen else (W, out.size(2))):
            raise ValueError("locations must be [W, S], or [total_q] with cu_seqlens_q")
        if varlen and tuple(cu_seqlens_q.shape) != (W + 1,):
            raise ValueError("cu_seqlens_q must be [W + 1]")
        if lse is not None and (lse.shape != out.shape[:-1] or lse.dtype != torch.float32):
            raise ValueError("lse must be float32 [W, Hq, S], or [total_q, Hq] with cu_seqlens_q")
        if any(t.dtype != torch.int32 for t in (locations, block_table) + ((cu_seqlens_q,) if varlen else ())):
            raise ValueError("locations, block_table and cu_seqlens_q must be int32")
        if any(t.dtype != out.dtype for t in (q, key_cache, value_cache)):
            raise ValueError("queries and caches must have the dtype of the output")
        if not 1 <= int(window) < 1 << 31 or not 0 <= int(sinks) < 1 << 31:
            raise ValueError("window must be positive and sinks not negative")
        tensors = [t for t in (out, q, locations, key_cache, value_cache, block_table, cu_seqlens_q, lse) if t is not None]
        for t in tensors:
            if not t.is_contiguous() or t.device != out.device:
                raise ValueError("all tensors must be contiguous and live on the output's device")
        self._keep, self.device, self.varlen = tensors, out.device, varlen
        p = HwWindowProblem()
        p.dtype = _DTYPE_CODE[out.dtype]
        p.W, p.Hq, p.Hkv, p.D = W, out.size(1), key_cache.size(1), key_cache.size(3)
        p.S, p.total_q = (0, out.size(0)) if varlen else (out.size(2), 0)
        p.block_size, p.max_blocks, p.num_blocks = key_cache.size(2), block_table.size(1), key_cache.size(0)
        p.window, p.sinks, p.scale = int(window), int(sinks), float(scale)
        p.out, p.q, p.locations = out.data_ptr(), q.data_ptr(), locations.data_ptr()
        p.lse = lse.data_ptr() if lse is not None else None
        p.key_cache, p.value_cache, p.block_table = key_cache.data_ptr(), value_cache.data_ptr(), block_table.data_ptr()
        p.cu_seqlens_q = cu_seqlens_q.data_ptr() if varlen else None
        p.splits, p.row_blocks = int(splits), int(row_blocks)
        self.p = p

    def run(self) -> None:
        with torch.cuda.device(self.device):
            n = C.c_size_t(0)
            check(lib.hw_window_workspace_bytes(C.byref(self.p), C.byref(n)), "hw_window_workspace_bytes")
            ws = torch.empty(n.value, dtype=torch.uint8, device=self.device) if n.value else None
            self.p.workspace, self.p.workspace_bytes = ws.data_ptr() if ws is not None else None, n.value
            fn = lib.hw_window_varlen_paged_sdpa if self.varlen else lib.hw_window_paged_sdpa
            check(fn(C.byref(self.p), C.c_void_p(torch.cuda.current_stream(self.device).cuda_stream)), fn.__name__)


def window_plan(*, W: int, Hq: int, Hkv: int, D: int, block_size: int, max_blocks: int, window: int, num_cus: int, sinks: int = 0, S: int = 0,
                total_q: Optional[int] = None, splits: int = 0, dtype: int = HW_BF16, row_blocks: int = 0) -> HwPagedPlan:
    """Host-only plan of the operators with a sliding window (no GPU needed); total_q selects the variable-length operator."""
    p = HwWindowProblem()
    p.dtype = dtype
    p.W, p.Hq, p.Hkv, p.D, p.S = W, Hq, Hkv, D, S
    p.block_size, p.max_blocks, p.num_blocks = block_size, max_blocks, 1
    p.window, p.sinks, p.scale = window, sinks, 1.0
    p.out = p.q = p.locations = p.key_cache = p.value_cache = p.block_table = 16       # only tested for being aligned and non-NULL
    if total_q is not None:
        p.total_q = total_q
        p.cu_seqlens_q = 16
    p.splits, p.row_blocks = splits, row_blocks
    out = HwPagedPlan()
    check(lib.hw_window_plan_debug(C.byref(p), num_cus, C.byref(out)), "hw_window_plan_debug")
    return out


def packed_slots(block_table: torch.Tensor, positions: torch.Tensor, n_new: torch.Tensor, cu_seqlens: torch.Tensor, locations: torch.Tensor,
                 slots: torch.Tensor, block_size: int, num_blocks: int) -> None:
    """cu_seqlens [W + 1], locations [total] and slots [total] of a packed batch, int32."""
    if block_table.dim() != 2 or block_table.numel() == 0 or tuple(positions.shape) != (block_table.size(0),) or positions.shape != n_new.shape:
        raise ValueError("block_table must be [W, max_blocks], positions and n_new [W]")
    W, total, block_size, num_blocks = block_table.size(0), locations.numel(), int(block_size), int(num_blocks)
    if tuple(cu_seqlens.shape) != (W + 1,) or tuple(locations.shape) != (total,) or slots.shape != locations.shape:
        raise ValueError("cu_seqlens must be [W + 1], locations and slots [total]")
    for t in (block_table, positions, n_new, cu_seqlens, locations, slots):
        if t.dtype != torch.int32 or not t.is_contiguous() or t.device != block_table.device:
            raise ValueError("the tables of a packed batch must be contiguous int32 on one device")
    if total >= 1 << 28 or not 1 <= block_size < 1 << 31 or not 1 <= num_blocks < 1 << 31:
        raise ValueError("total must be below 2^28, block_size and num_blocks positive")
    b = HwPackedBatch(W, block_table.size(1), num_blocks, block_size, total, block_table.data_ptr(), positions.data_ptr(), n_new.data_ptr(),
                      cu_seqlens.data_ptr(), locations.data_ptr(), slots.data_ptr())
    with torch.cuda.device(block_table.device):
        check(lib.hw_packed_slots(C.byref(b), C.c_void_p(torch.cuda.current_stream(block_table.device).cuda_stream)), "hw_packed_slots")


def copy_to_slots(key_states: torch.Tensor, value_states: torch.Tensor, key_cache: torch.Tensor, value_cache: torch.Tensor, slots: torch.Tensor) -> None:
    """Rows [total, Hkv, E|Ev] (any strides with a contiguous last dimension) to the rows `slots` of the paged caches."""
    if key_states.dim() != 3 or value_states.dim() != 3 or key_states.shape[:2] != value_states.shape[:2]:
        raise ValueError("key_states / value_states must be [total, Hkv, E|Ev]")
    T, Hkv, E = key_states.shape
    Ev = value_states.size(2)
    if key_cache.dim() != 4 or value_cache.dim() != 4 or key_cache.size(1) != Hkv or key_cache.shape[:3] != value_cache.shape[:3] \
            or key_cache.size(3) != E or value_cache.size(3) != Ev or not key_cache.is_contiguous() or not value_cache.is_contiguous():
        raise ValueError("caches must be contiguous [num_blocks, Hkv, block_size, E|Ev] and match the states")
    if key_states.dtype not in _DTYPE_CODE:
        raise HogwildError(-2, "copy_to_slots")
    if any(t.dtype != key_states.dtype for t in (value_states, key_cache, value_cache)):
        raise ValueError("states and caches must share one dtype")
    if tuple(slots.shape) != (T,) or slots.dtype != torch.int32 or not slots.is_contiguous():
        raise ValueError("slots must be contiguous int32 [total]")
    if any(t.device != key_cache.device for t in (key_states, value_states, value_cache, slots)):
        raise ValueError("all tensors must live on the caches' device")
    if (E > 1 and key_states.stride(2) != 1) or (Ev > 1 and value_states.stride(2) != 1):
        key_states, value_states = key_states.contiguous(), value_states.contiguous()
    c = HwCopySlots(_DTYPE_CODE[key_states.dtype], T, Hkv, E, Ev, key_cache.size(2), key_cache.size(0), key_states.data_ptr(), value_states.data_ptr(),
                    key_states.stride(0), key_states.stride(1), value_states.stride(0), value_states.stride(1), key_cache.data_ptr(),
                    value_cache.data_ptr(), slots.data_ptr())
    with torch.cuda.device(key_cache.device):
        check(lib.hw_copy_to_slots(C.byref(c), C.c_void_p(torch.cuda.current_stream(key_cache.device).cuda_stream)), "hw_copy_to_slots")


def verify_drafts(drafts: torch.Tensor, target_probs: torch.Tensor, uniforms: torch.Tensor, draft_probs: Optional[torch.Tensor] = None,
                  n_drafts: Optional[torch.Tensor] = None, positions: Optional[torch.Tensor] = None, seq_lengths: Optional[torch.Tensor] = None,
                  n_new: Optional[torch.Tensor] = None):
    """(tokens [W, K + 1], accepted int32 [W]) of drafts [W, K]; see hw_verify."""
    if drafts.dim() != 2 or drafts.dtype not in (torch.int32, torch.int64) or not drafts.is_contiguous():
        raise ValueError("drafts must be contiguous int64 or int32 [W, K]")
    W, K = drafts.shape
    if target_probs.dim() != 3 or tuple(target_probs.shape[:2]) != (W, K + 1) or target_probs.size(2) < 1:
        raise ValueError("target_probs must be [W, K + 1, V]")
    V = target_probs.size(2)
    if target_probs.dtype not in _DTYPE_CODE:
        raise HogwildError(-2, "verify_drafts")
    if tuple(uniforms.shape) != (W, K + 1) or uniforms.dtype != torch.float32 or not uniforms.is_contiguous():
        raise ValueError("uniforms must be contiguous float32 [W, K + 1]")
    if draft_probs is not None and (tuple(draft_probs.shape) != (W, K, V) or draft_probs.dtype != target_probs.dtype):
        raise ValueError("draft_probs must be [W, K, V] in the dtype of target_probs")
    if (positions is None) != (seq_lengths is None):
        raise ValueError("positions and seq_lengths go together")
    if n_new is not None and seq_lengths is None:
        raise ValueError("n_new goes with positions and seq_lengths")
    for t in (n_drafts, positions, seq_lengths, n_new):
        if t is not None and (tuple(t.shape) != (W,) or t.dtype != torch.int32 or not t.is_contiguous()):
            raise ValueError("n_drafts, positions, seq_lengths and n_new must be contiguous int32 [W]")
    device = target_probs.device
    if any(t is not None and t.device != device for t in (drafts, uniforms, draft_probs, n_drafts, positions, seq_lengths, n_new)):
        raise ValueError("all tensors must live on one device")
    if V > 1 and target_probs.stride(2) != 1:
        target_probs = target_probs.contiguous()
    if draft_probs is not None and V > 1 and draft_probs.stride(2) != 1:
        draft_probs = draft_probs.contiguous()
    tokens, accepted = torch.empty((W, K + 1), dtype=drafts.dtype, device=device), torch.empty(W, dtype=torch.int32, device=device)
    ptr = lambda t: t.data_ptr() if t is not None else None      # noqa: E731
    v = HwVerify()
    v.dtype, v.token_bytes = _DTYPE_CODE[target_probs.dtype], drafts.element_size()
    v.W, v.K, v.V = W, K, V
    v.drafts, v.target, v.draft_probs = drafts.data_ptr(), target_probs.data_ptr(), ptr(draft_probs) if K else None
    v.tp_w, v.tp_k = target_probs.stride(0), target_probs.stride(1)
    if draft_probs is not None:
        v.dp_w, v.dp_k = draft_probs.stride(0), draft_probs.stride(1)
    v.uniforms, v.n_drafts, v.positions, v.seq_lengths = uniforms.data_ptr(), ptr(n_drafts), ptr(positions), ptr(seq_lengths)
    v.n_new = ptr(n_new)
    v.tokens, v.accepted = tokens.data_ptr(), accepted.data_ptr()
    with torch.cuda.device(device):
        n = C.c_size_t(0)
        check(lib.hw_verify_workspace_bytes(C.byref(v), C.byref(n)), "hw_verify_workspace_bytes")
        ws = torch.empty(n.value, dtype=torch.uint8, device=device) if n.value else None
        v.workspace, v.workspace_bytes = ptr(ws), n.value
        check(lib.hw_verify_drafts(C.byref(v), C.c_void_p(torch.cuda.current_stream(device).cuda_stream)), "hw_verify_drafts")
    return tokens, accepted


class _Pool:
    """hw_pool of a block table [W, max_blocks], the sequences' lengths [W], the pages' counts [num_blocks] and the caches."""

    def __init__(self, block_table: torch.Tensor, seq_lengths: Optional[torch.Tensor], ref_counts: torch.Tensor, block_size: int = 1,
                 caches: Sequence[torch.Tensor] = ()):
        if block_table.dim() != 2 or ref_counts.dim() != 1 or block_table.numel() == 0 or ref_counts.numel() == 0:
            raise ValueError("block_table must be [W, max_blocks], ref_counts [num_blocks]")
        if seq_lengths is not None and tuple(seq_lengths.shape) != (block_table.size(0),):
            raise ValueError("seq_lengths must be [W]")
        if int(block_size) < 1:
            raise ValueError("block_size must be positive")
        self.device = block_table.device
        self.vectors = [t for t in (block_table, seq_lengths, ref_counts) if t is not None]
        self.check_ints(*self.vectors)
        p = HwPool()
        p.W, p.max_blocks, p.num_blocks, p.block_size = block_table.size(0), block_table.size(1), ref_counts.numel(), int(block_size)
        p.block_table, p.ref_counts = block_table.data_ptr(), ref_counts.data_ptr()
        p.seq_lengths = seq_lengths.data_ptr() if seq_lengths is not None else None
        self._ptr, self._bytes = _pages_of(caches, p.num_blocks, self.device)
        p.caches, p.page_bytes, p.n_caches = C.cast(self._ptr, C.POINTER(C.c_void_p)), C.cast(self._bytes, C.POINTER(C.c_size_t)), len(caches)
        self.p = p

    def check_ints(self, *tensors: torch.Tensor) -> None:
        for t in tensors:
            if t.dtype != torch.int32 or not t.is_contiguous() or t.device != self.device:
                raise ValueError("the tables of a pool must be contiguous int32 on one device")

    def run(self, fn, *args, workspace: bool = False) -> None:
        with torch.cuda.device(self.device):
            if workspace:
                n = C.c_size_t(0)
                check(lib.hw_pool_workspace_bytes(C.byref(self.p), C.byref(n)), "hw_pool_workspace_bytes")
                ws = torch.empty(n.value, dtype=torch.uint8, device=self.device)
                self.p.workspace, self.p.workspace_bytes = ws.data_ptr(), n.value
            stream = torch.cuda.current_stream(self.device).cuda_stream
            check(fn(C.byref(self.p), *args, C.c_void_p(stream)), fn.__name__)


def _pages_of(caches: Sequence[torch.Tensor], num_blocks: int, device):
    for i, t in enumerate(caches):
        if t.dim() < 1 or t.size(0) != num_blocks or not t.is_contiguous() or t.numel() == 0 or t.device != device:
            raise ValueError(f"cache {i} must be contiguous [num_blocks, ...] with {num_blocks} blocks on the pool's device")
    n = max(1, len(caches))
    return ((C.c_void_p * n)(*[t.data_ptr() for t in caches]),
            (C.c_size_t * n)(*[t.numel() // num_blocks * t.element_size() for t in caches]))


def fork_blocks(block_table, seq_lengths, ref_counts, parents, block_size: int) -> None:
    pool = _Pool(block_table, seq_lengths, ref_counts, block_size)
    if tuple(parents.shape) != (block_table.size(0),):
        raise ValueError("parents must be [W]")
    pool.check_ints(parents)
    pool.run(lib.hw_fork_blocks, parents.data_ptr())


def free_blocks(block_table, seq_lengths, ref_counts, finished) -> None:
    pool = _Pool(block_table, seq_lengths, ref_counts)
    if tuple(finished.shape) != (block_table.size(0),) or finished.dtype not in (torch.bool, torch.uint8) or not finished.is_contiguous() \
            or finished.device != pool.device:
        raise ValueError("finished must be contiguous bool [W]")
    pool.run(lib.hw_free_blocks, finished.data_ptr())


def trim_blocks(block_table, seq_lengths, ref_counts, window: int, sinks: int, block_size: int) -> None:
    if not 1 <= int(window) < 1 << 31 or not 0 <= int(sinks) < 1 << 31:
        raise ValueError("window must be positive and sinks not negative")
    _Pool(block_table, seq_lengths, ref_counts, block_size).run(lib.hw_trim_blocks, int(window), int(sinks))


def reserve_blocks(block_table, seq_lengths, ref_counts, n_new, positions, caches, block_size: int, total: int = -1) -> None:
    pool = _Pool(block_table, seq_lengths, ref_counts, block_size, caches)
    W = block_table.size(0)
    if tuple(n_new.shape) != (W,) or tuple(positions.shape) not in ((W,), (2, W)):
        raise ValueError("n_new must be [W], positions [W] or [2, W]")
    if total != -1 and not (positions.dim() == 2 and 0 <= int(total) < 1 << 28):
        raise ValueError("the rows of a packed batch are below 2^28, and go with positions [2, W]")
    pool.check_ints(n_new, positions)
    if positions.dim() == 2:
        pool.run(lib.hw_reserve_step, n_new.data_ptr(), int(total), positions.data_ptr(), positions[1].data_ptr(), workspace=True)
    else:
        pool.run(lib.hw_reserve_blocks, n_new.data_ptr(), positions.data_ptr(), workspace=True)


def compact_blocks(block_table, ref_counts, caches, used) -> None:
    pool = _Pool(block_table, None, ref_counts, 1, caches)
    if used.numel() != 1:
        raise ValueError("used must be one number")
    pool.check_ints(used)
    pool.run(lib.hw_compact_blocks, used.data_ptr(), workspace=True)


def capture_id(device: torch.device) -> int:
    """A number of its own for the graph capture that the device's current stream is in, 0 outside of any."""
    if device.index != torch.cuda.current_device():
        with torch.cuda.device(device):
            return capture_id(device)
    if not torch.cuda.is_current_stream_capturing():
        return 0
    n = C.c_ulonglong(0)
    check(lib.hw_stream_capture_id(C.c_void_p(torch.cuda.current_stream(device).cuda_stream), C.byref(n)), "hw_stream_capture_id")
    return n.value


def copy_blocks(caches: Sequence[torch.Tensor], src: Sequence[int], dst: Sequence[int]) -> None:
    if len(caches) == 0 or caches[0].dim() < 1:
        raise ValueError("copy_blocks needs caches [num_blocks, ...]")
    if len(src) != len(dst):
        raise ValueError("one destination for every source block")
    nb, device = caches[0].size(0), caches[0].device
    if any(not 0 <= int(x) < nb for x in list(src) + list(dst)):
        raise ValueError(f"blocks outside 0..{nb - 1}")
    ptr, nbytes = _pages_of(caches, nb, device)
    n = len(src)
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        check(lib.hw_copy_pages(ptr, nbytes, len(caches), nb, (C.c_int32 * max(1, n))(*[int(x) for x in src]),
                                (C.c_int32 * max(1, n))(*[int(x) for x in dst]), n, C.c_void_p(stream)), "hw_copy_pages")


def build_inputs(pos_end: Sequence[Sequence[int]], S: int, inv_freq: Optional[torch.Tensor], *, attention_scaling: float = 1.0,
                 table_dtype: Optional[torch.dtype] = None, device=None):
    """locations int32 [F, W, S], cosines / sines float32 [F, W, S, RotE] of a decode step.  pos_end[f][w] = position one
    past the newest token of worker w as seen through fragment f (host numbers).  table_dtype = dtype the tables are
    rounded to before being stored as float32 (None / float32: no rounding)."""
    F, W = len(pos_end), len(pos_end[0])
    flat = [int(x) for row in pos_end for x in row]
    if len(flat) != F * W:
        raise ValueError("pos_end must be a full [F][W] table")
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    if inv_freq is not None:
        if inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous():
            raise ValueError("inv_freq must be contiguous float32 [RotE/2]")
        device = inv_freq.device
    if device is None:
        raise ValueError("a device is needed when there is no inv_freq tensor")
    device = torch.device(device)
    loc = torch.empty((F, W, S), dtype=torch.int32, device=device)
    cos = torch.empty((F, W, S, rot), dtype=torch.float32, device=device)
    sin = torch.empty((F, W, S, rot), dtype=torch.float32, device=device)
    arr = (C.c_int32 * (F * W))(*flat)
    rd = HW_F32 if table_dtype is None else _DTYPE_CODE[table_dtype]
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        check(lib.hw_build_inputs(loc.data_ptr(), cos.data_ptr(), sin.data_ptr(), arr,
                                  inv_freq.data_ptr() if inv_freq is not None else None, float(attention_scaling), rd,
                                  F, W, S, rot, C.c_void_p(stream)), "hw_build_inputs")
    return loc, cos, sin


def build_inputs_dev(len_dev: torch.Tensor, orders: Sequence[Sequence[int]], S: int, inv_freq: Optional[torch.Tensor], *,
                     attention_scaling: float = 1.0, table_dtype: Optional[torch.dtype] = None, out=None):
    """build_inputs with the fragment lengths in device memory: len_dev int32 [F] (lengths including this step's new
    tokens), orders[w] = the fragments in worker w's order.  out = (locations, cosines, sines) to write into (so that a
    captured graph keeps its addresses), else fresh tensors."""
    F, W = len_dev.numel(), len(orders)
    flat = [int(x) for row in orders for x in row]
    if len(flat) != F * W:
        raise ValueError("every worker's order must list all F fragments")
    if len_dev.dtype != torch.int32 or not len_dev.is_contiguous():
        raise ValueError("len_dev must be contiguous int32 [F]")
    device = len_dev.device
    rot = 0 if inv_freq is None else 2 * inv_freq.numel()
    if inv_freq is not None and (inv_freq.dtype != torch.float32 or not inv_freq.is_contiguous() or inv_freq.device != device):
        raise ValueError("inv_freq must be contiguous float32 [RotE/2] on the device of len_dev")
    if out is None:
        out = (torch.empty((F, W, S), dtype=torch.int32, device=device), torch.empty((F, W, S, rot), dtype=torch.float32, device=device),
               torch.empty((F, W, S, rot), dtype=torch.float32, device=device))
    loc, cos, sin = out
    if tuple(loc.shape) != (F, W, S) or loc.dtype != torch.int32 or tuple(cos.shape) != (F, W, S, rot) or tuple(sin.shape) != (F, W, S, rot) \
            or cos.dtype != torch.float32 or sin.dtype != torch.float32 or not (loc.is_contiguous() and cos.is_contiguous() and sin.is_contiguous()):
        raise ValueError("out must be (int32 [F, W, S], float32 [F, W, S, RotE], float32 [F, W, S, RotE]), contiguous")
    arr = (C.c_int32 * (F * W))(*flat)
    rd = HW_F32 if table_dtype is None else _DTYPE_CODE[table_dtype]
    with torch.cuda.device(device):
        stream = torch.cuda.current_stream(device).cuda_stream
        check(lib.hw_build_inputs_dev(loc.data_ptr(), cos.data_ptr(), sin.data_ptr(), len_dev.data_ptr(), arr,
                                      inv_freq.data_ptr() if inv_freq is not None else None, float(attention_scaling), rd,
                                      F, W, S, rot, C.c_void_p(stream)), "hw_build_inputs_dev")
    return loc, cos, sin


def advance_lengths(len_dev: torch.Tensor, add: Sequence[int]) -> None:
    """len_dev[f] += add[f] on the device (add: host numbers)."""
    F = len_dev.numel()
    if len_dev.dtype != torch.int32 or not len_dev.is_contiguous() or len(add) != F:
        raise ValueError("len_dev must be contiguous int32 [F] and add one number per entry")
    arr = (C.c_int32 * F)(*[int(x) for x in add])
    with torch.cuda.device(len_dev.device):
        stream = torch.cuda.current_stream(len_dev.device).cuda_stream
        check(lib.hw_advance_lengths(len_dev.data_ptr(), arr, F, C.c_void_p(stream)), "hw_advance_lengths")


def rope_append(key_states: torch.Tensor, value_states: torch.Tensor, k_dst: Sequence[torch.Tensor], v_dst: Sequence[torch.Tensor],
                dst_len: Sequence[int], *, cosines: Optional[torch.Tensor] = None, sines: Optional[torch.Tensor] = None,
                n_new: Optional[Sequence[int]] = None, mode: int = HW_ROPE_EAGER, len_dev: Optional[torch.Tensor] = None) -> None:
    """Rotate key_states [W, Hkv, S, E] with cosines / sines [W, S, RotE] (or [W, 1, RotE]: one row for all tokens) and
    append keys and value_states [W, Hkv, S, Ev] to the segment buffers k_dst[w] / v_dst[w] ([Hkv, cap, E|Ev], contiguous)
    behind their first dst_len[w] rows.  Without cosines the keys are appended as they are.  n_new[w] < S appends only
    the last n_new[w] tokens of worker w.  With len_dev (int32 device tensor of segment lengths) dst_len[w] is an index
    into it and len_dev[dst_len[w]] the length of worker w's segment after this append."""
    if key_states.dim() != 4 or value_states.dim() != 4 or key_states.shape[:3] != value_states.shape[:3]:
        raise ValueError("key_states / value_states must be [W, Hkv, S, E|Ev]")
    W, Hkv, S, E = key_states.shape
    Ev = value_states.size(3)
    if key_states.dtype not in _DTYPE_CODE or value_states.dtype != key_states.dtype:
        raise HogwildError(-2, "rope_append")
    if (E > 1 and key_states.stride(3) != 1) or (Ev > 1 and value_states.stride(3) != 1):
        key_states, value_states = key_states.contiguous(), value_states.contiguous()
    if len(k_dst) != W or len(v_dst) != W or len(dst_len) != W:
        raise ValueError("one destination segment and length per worker")
    for kd, vd in zip(k_dst, v_dst):
        if kd.dim() != 3 or vd.dim() != 3 or kd.size(0) != Hkv or vd.size(0) != Hkv or kd.size(2) != E or vd.size(2) != Ev \
                or kd.size(1) != vd.size(1) or not kd.is_contiguous() or not vd.is_contiguous():
            raise ValueError("segment buffers must be contiguous [Hkv, cap, E|Ev] with one capacity for keys and values")
        if kd.dtype != key_states.dtype or vd.dtype != key_states.dtype or kd.device != key_states.device:
            raise ValueError("segment buffers must have the dtype and device of the new states")
    a = HwAppend()
    a.dtype = _DTYPE_CODE[key_states.dtype]
    a.mode = int(mode)
    a.W, a.Hkv, a.S, a.E, a.Ev = W, Hkv, S, E, Ev
    a.key_states, a.value_states = key_states.data_ptr(), value_states.data_ptr()
    a.ks_w, a.ks_h, a.ks_s = key_states.stride(0), key_states.stride(1), key_states.stride(2)
    a.vs_w, a.vs_h, a.vs_s = value_states.stride(0), value_states.stride(1), value_states.stride(2)
    a.cs_dtype = HW_F32
    keep = [key_states, value_states]
    if cosines is not None:
        if sines is None or cosines.shape != sines.shape or cosines.dim() != 3 or cosines.size(0) != W or cosines.size(1) not in (1, S):
            raise ValueError("cosines / sines must be [W, S, RotE] or [W, 1, RotE]")
        if cosines.dtype != sines.dtype or cosines.dtype not in (torch.float32, key_states.dtype):
            raise ValueError("cosines / sines must be float32 or have the dtype of the keys")
        cosines, sines = cosines.contiguous(), sines.contiguous()
        a.RotE = cosines.size(2)
        a.cs_dtype = _DTYPE_CODE[cosines.dtype]
        a.cosines, a.sines = cosines.data_ptr(), sines.data_ptr()
        a.cs_w = cosines.stride(0)
        a.cs_s = 0 if cosines.size(1) == 1 else cosines.stride(1)
        keep += [cosines, sines]
    kp = (C.c_void_p * W)(*[t.data_ptr() for t in k_dst])
    vp = (C.c_void_p * W)(*[t.data_ptr() for t in v_dst])
    ln = (C.c_int32 * W)(*[int(x) for x in dst_len])
    cp = (C.c_int32 * W)(*[t.size(1) for t in k_dst])
    nn = (C.c_int32 * W)(*([S] * W if n_new is None else [int(x) for x in n_new]))
    a.k_dst, a.v_dst = C.cast(kp, C.POINTER(C.c_void_p)), C.cast(vp, C.POINTER(C.c_void_p))
    a.dst_len, a.dst_cap, a.n_new = C.cast(ln, C.POINTER(C.c_int32)), C.cast(cp, C.POINTER(C.c_int32)), C.cast(nn, C.POINTER(C.c_int32))
    if len_dev is not None:
        if len_dev.dtype != torch.int32 or len_dev.dim() != 1 or not len_dev.is_contiguous() or len_dev.device != key_states.device:
            raise ValueError("len_dev must be a contiguous int32 vector on the device of the new states")
        if any(int(x) < 0 or int(x) >= len_dev.numel() for x in dst_len):
            raise ValueError("with len_dev, dst_len holds indices into it")
        a.len_dev = len_dev.data_ptr()
    with torch.cuda.device(key_states.device):
        stream = torch.cuda.current_stream(key_states.device).cuda_stream
        check(lib.hw_rope_append(C.byref(a), C.c_void_p(stream)), "hw_rope_append")


class AppendPlan:
    """hw_rope_append with everything that stays the same from step to step prepared once: destination buffers,
    capacities, tokens per worker, and the segment lengths in device memory.  run() fills in the new states and their
    rotary tables and launches; it checks only what can change between calls."""

    def __init__(self, k_dst: Sequence[torch.Tensor], v_dst: Sequence[torch.Tensor], seg_index: Sequence[int], n_new: Sequence[int],
                 len_dev: torch.Tensor, mode: int = HW_ROPE_EAGER):
        W = len(k_dst)
        if len(v_dst) != W or len(seg_index) != W or len(n_new) != W:
            raise ValueError("one destination segment, length index and token count per worker")
        kd0 = k_dst[0]
        for kd, vd in zip(k_dst, v_dst):
            if kd.dim() != 3 or vd.dim() != 3 or kd.shape[:2] != vd.shape[:2] or not kd.is_contiguous() or not vd.is_contiguous() \
                    or kd.size(0) != kd0.size(0) or kd.size(2) != kd0.size(2) or vd.size(2) != v_dst[0].size(2) \
                    or kd.dtype != kd0.dtype or vd.dtype != kd0.dtype or kd.device != kd0.device:
                raise ValueError("segment buffers must be contiguous [Hkv, cap, E|Ev] of one dtype on one device")
        if len_dev.dtype != torch.int32 or len_dev.dim() != 1 or not len_dev.is_contiguous() or len_dev.device != kd0.device:
            raise ValueError("len_dev must be a contiguous int32 vector on the device of the segments")
        if any(int(x) < 0 or int(x) >= len_dev.numel() for x in seg_index):
            raise ValueError("seg_index holds indices into len_dev")
        self.W, self.Hkv, self.E, self.Ev = W, kd0.size(0), kd0.size(2), v_dst[0].size(2)
        self.dtype, self.device = kd0.dtype, kd0.device
        self._keep = (list(k_dst), list(v_dst), len_dev)
        self._kp = (C.c_void_p * W)(*[t.data_ptr() for t in k_dst])
        self._vp = (C.c_void_p * W)(*[t.data_ptr() for t in v_dst])
        self._ln = (C.c_int32 * W)(*[int(x) for x in seg_index])
        self._cp = (C.c_int32 * W)(*[t.size(1) for t in k_dst])
        self._nn = (C.c_int32 * W)(*[int(x) for x in n_new])
        a = HwAppend()
        a.dtype = _DTYPE_CODE[self.dtype]
        a.mode = int(mode)
        a.W, a.Hkv, a.E, a.Ev = W, self.Hkv, self.E, self.Ev
        a.k_dst, a.v_dst = C.cast(self._kp, C.POINTER(C.c_void_p)), C.cast(self._vp, C.POINTER(C.c_void_p))
        a.dst_len, a.dst_cap, a.n_new = (C.cast(self._ln, C.POINTER(C.c_int32)), C.cast(self._cp, C.POINTER(C.c_int32)),
                                         C.cast(self._nn, C.POINTER(C.c_int32)))
        a.len_dev = len_dev.data_ptr()
        self.a = a

    def run(self, key_states: torch.Tensor, value_states: torch.Tensor, cosines: Optional[torch.Tensor] = None,
            sines: Optional[torch.Tensor] = None) -> None:
        a = self.a
        W, Hkv, S, E = key_states.shape
        if (W, Hkv, E) != (self.W, self.Hkv, self.E) or tuple(value_states.shape) != (W, Hkv, S, self.Ev) \
                or key_states.dtype != self.dtype or value_states.dtype != self.dtype or key_states.device != self.device:
            raise ValueError("new states do not match the prepared append")
        if (E > 1 and key_states.stride(3) != 1) or (self.Ev > 1 and value_states.stride(3) != 1):
            key_states, value_states = key_states.contiguous(), value_states.contiguous()
        a.S = S
        a.key_states, a.value_states = key_states.data_ptr(), value_states.data_ptr()
        a.ks_w, a.ks_h, a.ks_s = key_states.stride(0), key_states.stride(1), key_states.stride(2)
        a.vs_w, a.vs_h, a.vs_s = value_states.stride(0), value_states.stride(1), value_states.stride(2)
        if cosines is None:
            a.RotE, a.cs_dtype, a.cosines, a.sines = 0, HW_F32, None, None
        else:
            if sines is None or cosines.shape != sines.shape or cosines.dim() != 3 or cosines.size(0) != W or cosines.size(1) not in (1, S) \
                    or cosines.dtype != sines.dtype or cosines.dtype not in (torch.float32, self.dtype):
                raise ValueError("cosines / sines must be [W, S, RotE] or [W, 1, RotE], float32 or in the dtype of the keys")
            cosines, sines = cosines.contiguous(), sines.contiguous()
            a.RotE = cosines.size(2)
            a.cs_dtype = _DTYPE_CODE[cosines.dtype]
            a.cosines, a.sines = cosines.data_ptr(), sines.data_ptr()
            a.cs_w = cosines.stride(0)
            a.cs_s = 0 if cosines.size(1) == 1 else cosines.stride(1)
        stream = torch.cuda.current_stream(self.device).cuda_stream
        check(lib.hw_rope_append(C.byref(a), C.c_void_p(stream)), "hw_rope_append")


def rope(q: torch.Tensor, cosines: torch.Tensor, sines: torch.Tensor, out: torch.Tensor) -> torch.Tensor:
    F, W, Hq, S, E = out.shape
    if tuple(q.shape) != (W, Hq, S, E) or q.dtype != out.dtype:
        raise ValueError("queries must be [W, Hq, S, E] in the output dtype")
    rot = cosines.size(-1)
    if tuple(cosines.shape) != (F, W, S, rot) or tuple(sines.shape) != (F, W, S, rot):
        raise ValueError("cosines / sines must be [F, W, S, RotE]")
    if cosines.dtype != torch.float32 or sines.dtype != torch.float32:
        raise ValueError("cosines / sines must be float32")
    for t in (q, cosines, sines, out):
        if not t.is_contiguous():
            raise ValueError("all tensors must be contiguous")
    with torch.cuda.device(out.device):
        stream = torch.cuda.current_stream(out.device).cuda_stream
        check(lib.hw_rope(out.data_ptr(), q.data_ptr(), cosines.data_ptr(), sines.data_ptr(), _DTYPE_CODE[out.dtype],
                          F, W, Hq, S, E, rot, C.c_void_p(stream)), "hw_rope")
    return out
