"""Python host-side mirror of the llm.c-style launcher surface, bound over the
C ABI of ``libgpt2_mi355x.so`` (declared in ``include/gpt2_mi355x.h``).

The launchers keep the reference's names and argument order
(``matmul_forward(out, inp, weight, bias, B, T, C, OC)`` and so on: reference
``kernels/matmul/2_matmul_cublas.cuh:34-42``,
``kernels/attention/3_flash_attention_permute.cuh:346-351``,
``kernels/fused_residual_layernorm/fused_residual_layernorm.cuh:88-90``).
Arguments are torch CUDA tensors, used only as owners of device memory: the
library receives raw pointers.  There is no CPU fallback: if the shared library
is missing or no GPU is present, calls raise.
"""
from __future__ import annotations

import ctypes
import os
import subprocess
from typing import Optional

_HERE = os.path.dirname(os.path.abspath(__file__))
_ROOT = os.path.dirname(_HERE)
LIB_PATH = os.path.join(_HERE, "libgpt2_mi355x.so")
SOURCES = ("layernorm.hip", "elementwise.hip", "matmul.hip", "attention.hip", "paged.hip",
           "decode.hip", "gpt2.hip")
HIPCC_FLAGS = (
    "-O3", "--offload-arch=gfx950", "-std=c++17", "-fPIC", "-shared",
    # packed-fp32 VALU forms are switched off for every HIP translation unit
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
    # keep MFMA accumulators in ordinary VGPRs: the softmax reads them with VALU
    # instructions, and copies out of the accumulation registers would cost issue slots
    "-mllvm", "-amdgpu-mfma-vgpr-form",
)

EXPORTS = (
    "gpt2hip_last_error", "gpt2hip_set_stream", "gpt2hip_get_stream", "gpt2hip_set_workspace",
    "encoder_forward", "encoder_forward_status",
    "layernorm_forward", "layernorm_forward_status",
    "fused_residual_layernorm_forward", "fused_residual_layernorm_forward_status",
    "residual_forward", "residual_forward_status",
    "gelu_forward", "gelu_forward_status",
    "matmul_forward", "matmul_forward_status",
    "matmul_forward_gelu", "matmul_forward_gelu_status", "matmul_forward_probe_status",
    "matmul_forward_tile_shape",
    "matmul_forward_splitk_workspace", "matmul_forward_splitk_status",
    "matmul_forward_splitk_plan", "matmul_forward_splitk_forced_status",
    "matmul_forward_residual_status", "matmul_forward_first_columns",
    "attention_forward", "attention_forward_status",
    "kv_store_paged_status", "attention_decode_paged_workspace", "attention_decode_paged_status",
    "kv_evict_paged_status",
    "argmax_forward", "argmax_forward_status",
    "matmul_forward_argmax_workspace", "matmul_forward_argmax_status",
    "matmul_forward_argmax_noalloc_status",
    "gpt2_checkpoint_read_config", "gpt2_build_from_checkpoint",
    "gpt2_create", "gpt2_destroy", "gpt2_num_parameters", "gpt2_params_device",
    "gpt2_load_params_host", "gpt2_reserve", "gpt2_forward", "gpt2_forward_status",
    "gpt2_forward_device_status", "gpt2_forward_graph_status",
    "gpt2_prefill_status", "gpt2_decode_status", "gpt2_decode_sync_status", "gpt2_decode_options", "gpt2_decode_probe_status", "gpt2_decode_probe_size",
    "gpt2_step_logits", "gpt2_cache_length",
    "gpt2_forward_argmax_status", "gpt2_forward_sums_in_matmul",
    "gpt2_forward_profiled_status", "gpt2hip_profile_marker_overhead_us", "gpt2_logits", "gpt2_lnf", "gpt2_argmax_status",
    "gpt2hip_timer_create", "gpt2hip_timer_destroy", "gpt2hip_timer_start",
    "gpt2hip_timer_stop_ms",
)


def build(verbose: bool = False) -> str:
    """Compile every HIP source for gfx950 into ``libgpt2_mi355x.so`` (in-tree)."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    cmd = [hipcc, *HIPCC_FLAGS, "-I", os.path.join(_ROOT, "include"), "-o", LIB_PATH]
    cmd += [os.path.join(_HERE, "csrc", s) for s in SOURCES]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    noise = "is not a recognized feature for this target"
    err = "\n".join(l for l in proc.stderr.splitlines() if noise not in l)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}):\n{err}")
    if verbose and err.strip():
        print(err)
    build_example()
    return LIB_PATH


EXAMPLE_SRC = os.path.join(_HERE, "examples", "llmc_style_driver.cpp")
EXAMPLE_BIN = os.path.join(_HERE, "examples", "llmc_style_driver")


def build_example() -> str:
    """Compile the plain-C++ llm.c-style driver against the library's C ABI (host code only)."""
    hipcc = os.environ.get("HIPCC", "/opt/rocm/bin/hipcc")
    cmd = [hipcc, "-O2", "-std=c++17", EXAMPLE_SRC, "-I", os.path.join(_ROOT, "include"),
           "-L", _HERE, "-lgpt2_mi355x", "-Wl,-rpath,$ORIGIN/..", "-o", EXAMPLE_BIN]
    proc = subprocess.run(cmd, capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed on the example driver ({proc.returncode}):\n{proc.stderr}")
    return EXAMPLE_BIN


class GPT2Config(ctypes.Structure):
    _fields_ = [("max_seq_len", ctypes.c_int), ("vocab_size", ctypes.c_int),
                ("num_layers", ctypes.c_int), ("num_heads", ctypes.c_int),
                ("channels", ctypes.c_int)]


class GPT2PagedCache(ctypes.Structure):
    _fields_ = [("keys", ctypes.c_void_p), ("values", ctypes.c_void_p), ("table", ctypes.c_void_p),
                ("type", ctypes.c_int), ("num_pages", ctypes.c_int), ("page_size", ctypes.c_int),
                ("max_pages", ctypes.c_int), ("kv_heads", ctypes.c_int), ("head_size", ctypes.c_int)]


# order of the GPT2_PROF_* enum in the header
PROF_CATEGORIES = ("encoder", "layernorm", "matmul_qkv", "attention", "matmul_attproj",
                   "fused_residual_layernorm", "matmul_fc_gelu", "matmul_fcproj", "matmul_lmhead")

GPT2_124M = dict(max_seq_len=1024, vocab_size=50257, num_layers=12, num_heads=12, channels=768)
GPT2_350M = dict(max_seq_len=1024, vocab_size=50257, num_layers=24, num_heads=16, channels=1024)
GPT2_774M = dict(max_seq_len=1024, vocab_size=50257, num_layers=36, num_heads=20, channels=1280)    # "large"
GPT2_1558M = dict(max_seq_len=1024, vocab_size=50257, num_layers=48, num_heads=25, channels=1600)   # "XL"

_lib: Optional[ctypes.CDLL] = None


def lib() -> ctypes.CDLL:
    """The loaded C-ABI library.  Raises if it has not been built."""
    global _lib
    if _lib is None:
        if not os.path.exists(LIB_PATH):
            raise RuntimeError(
                f"{LIB_PATH} is missing: build it with __graft_entry__.build() "
                "(there is no CPU or PyTorch fallback for these kernels)")
        L = ctypes.CDLL(LIB_PATH)
        vp, ci, cz = ctypes.c_void_p, ctypes.c_int, ctypes.c_size_t
        L.gpt2hip_last_error.restype = ctypes.c_char_p
        sig = {
            "encoder_forward": [vp] * 4 + [ci] * 3,
            "layernorm_forward": [vp] * 6 + [ci] * 3,
            "fused_residual_layernorm_forward": [vp] * 8 + [ci] * 3,
            "residual_forward": [vp] * 3 + [ci],
            "gelu_forward": [vp] * 2 + [ci],
            "matmul_forward": [vp] * 4 + [ci] * 4,
            "matmul_forward_gelu": [vp] * 4 + [ci] * 5,
            "attention_forward": [vp] * 4 + [ci] * 4,
            "argmax_forward": [vp] * 2 + [ci] * 2,
        }
        for name, args in sig.items():
            f = getattr(L, name)
            f.argtypes, f.restype = args, None
            f = getattr(L, name + "_status")
            f.argtypes, f.restype = args, ci
        L.matmul_forward_probe_status.argtypes = [vp] * 4 + [ci] * 4 + [vp, ci, ctypes.POINTER(ci)]
        L.matmul_forward_probe_status.restype = ci
        L.matmul_forward_tile_shape.argtypes = [ci] * 4 + [ctypes.POINTER(ci)] * 2
        L.matmul_forward_tile_shape.restype = ci
        L.matmul_forward_splitk_workspace.argtypes = []
        L.matmul_forward_splitk_workspace.restype = cz
        L.matmul_forward_splitk_status.argtypes = [vp] * 4 + [ci] * 5 + [vp, cz]
        L.matmul_forward_splitk_status.restype = ci
        L.matmul_forward_splitk_forced_status.argtypes = [vp] * 4 + [ci] * 5 + [vp, cz] + [ci] * 3
        L.matmul_forward_splitk_forced_status.restype = ci
        L.matmul_forward_first_columns.argtypes = [ci] * 4 + [cz]
        L.matmul_forward_first_columns.restype = ci
        L.matmul_forward_residual_status.argtypes = [vp] * 5 + [ci] * 4 + [vp, cz]
        L.matmul_forward_residual_status.restype = ci
        L.matmul_forward_splitk_plan.argtypes = [ci] * 4 + [cz] + [ctypes.POINTER(ci)] * 3
        L.matmul_forward_splitk_plan.restype = ci
        L.kv_store_paged_status.argtypes = [vp, vp, ci, vp, vp, ci, ci, ci]
        L.kv_store_paged_status.restype = ci
        L.attention_decode_paged_workspace.argtypes = [vp, ci, ci, ci]
        L.attention_decode_paged_workspace.restype = cz
        L.attention_decode_paged_status.argtypes = [vp, vp, vp, ci] + [vp] * 3 + [ci] * 3 + [vp, cz]
        L.attention_decode_paged_status.restype = ci
        L.kv_evict_paged_status.argtypes = [vp] * 7 + [ci] * 3
        L.kv_evict_paged_status.restype = ci
        L.gpt2_create.argtypes, L.gpt2_create.restype = [ctypes.POINTER(GPT2Config)], vp
        L.gpt2_destroy.argtypes, L.gpt2_destroy.restype = [vp], None
        L.gpt2_checkpoint_read_config.argtypes = [ctypes.c_char_p, ctypes.POINTER(GPT2Config)]
        L.gpt2_checkpoint_read_config.restype = ci
        L.gpt2_build_from_checkpoint.argtypes = [ctypes.c_char_p]
        L.gpt2_build_from_checkpoint.restype = vp
        L.gpt2_num_parameters.argtypes, L.gpt2_num_parameters.restype = [vp], cz
        L.gpt2_params_device.argtypes, L.gpt2_params_device.restype = [vp], vp
        L.gpt2_load_params_host.argtypes, L.gpt2_load_params_host.restype = [vp, vp, cz], ci
        L.gpt2_reserve.argtypes, L.gpt2_reserve.restype = [vp, ci, ci], ci
        L.gpt2_forward.argtypes, L.gpt2_forward.restype = [vp, vp, ci, ci], None
        L.gpt2_forward_status.argtypes, L.gpt2_forward_status.restype = [vp, vp, ci, ci], ci
        L.gpt2_forward_device_status.argtypes = [vp, vp, ci, ci]
        L.gpt2_forward_device_status.restype = ci
        L.gpt2_prefill_status.argtypes, L.gpt2_prefill_status.restype = [vp, vp, ci, ci], ci
        L.gpt2_decode_status.argtypes, L.gpt2_decode_status.restype = [vp, vp], ci
        L.gpt2_decode_options.argtypes, L.gpt2_decode_options.restype = [vp, ci, ctypes.c_uint], ci
        L.gpt2_decode_sync_status.argtypes, L.gpt2_decode_sync_status.restype = [vp], ci
        L.gpt2_decode_probe_status.argtypes, L.gpt2_decode_probe_status.restype = [vp, vp, vp, cz], ci
        L.gpt2_decode_probe_size.argtypes, L.gpt2_decode_probe_size.restype = [vp], cz
        L.gpt2_step_logits.argtypes, L.gpt2_step_logits.restype = [vp], vp
        L.gpt2_cache_length.argtypes, L.gpt2_cache_length.restype = [vp], ci
        L.gpt2_forward_graph_status.argtypes = [vp, vp, ci, ci]
        L.gpt2_forward_graph_status.restype = ci
        L.gpt2hip_set_stream.argtypes, L.gpt2hip_set_stream.restype = [vp], None
        L.gpt2hip_get_stream.argtypes, L.gpt2hip_get_stream.restype = [], vp
        L.gpt2hip_set_workspace.argtypes, L.gpt2hip_set_workspace.restype = [vp, cz], ci
        L.gpt2_forward_sums_in_matmul.argtypes = [ctypes.POINTER(GPT2Config), ci, ci]
        L.gpt2_forward_sums_in_matmul.restype = ci
        L.gpt2_forward_argmax_status.argtypes = [vp, vp, ci, ci, vp]
        L.gpt2_forward_argmax_status.restype = ci
        L.matmul_forward_argmax_workspace.argtypes = [ci, ci, ci]
        L.matmul_forward_argmax_workspace.restype = cz
        L.matmul_forward_argmax_status.argtypes = [vp, vp, cz, vp, vp, vp, ci, ci, ci, ci]
        L.matmul_forward_argmax_status.restype = ci
        L.matmul_forward_argmax_noalloc_status.argtypes = [vp, vp, vp, vp, ci, ci, ci, ci]
        L.matmul_forward_argmax_noalloc_status.restype = ci
        L.gpt2_forward_profiled_status.argtypes = [vp, vp, ci, ci, ctypes.POINTER(ctypes.c_float)]
        L.gpt2_forward_profiled_status.restype = ci
        L.gpt2hip_profile_marker_overhead_us.argtypes = [ci]
        L.gpt2hip_profile_marker_overhead_us.restype = ctypes.c_float
        L.gpt2_logits.argtypes, L.gpt2_logits.restype = [vp], vp
        L.gpt2_lnf.argtypes, L.gpt2_lnf.restype = [vp], vp
        L.gpt2_argmax_status.argtypes, L.gpt2_argmax_status.restype = [vp, vp], ci
        L.gpt2hip_timer_create.argtypes, L.gpt2hip_timer_create.restype = [], vp
        L.gpt2hip_timer_destroy.argtypes, L.gpt2hip_timer_destroy.restype = [vp], None
        L.gpt2hip_timer_start.argtypes, L.gpt2hip_timer_start.restype = [vp], ci
        L.gpt2hip_timer_stop_ms.argtypes, L.gpt2hip_timer_stop_ms.restype = [vp], ctypes.c_float
        _lib = L
    return _lib


class GPT2HipError(RuntimeError):
    pass


def _check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().gpt2hip_last_error().decode(errors="replace")
        raise GPT2HipError(f"{what} failed (code {rc}): {msg}")


def _ptr(t, dtype=None) -> Optional[int]:
    """Device pointer of a contiguous CUDA tensor (None passes NULL)."""
    if t is None:
        return None
    import torch
    if not isinstance(t, torch.Tensor) or not t.is_cuda:
        raise TypeError("expected a CUDA tensor: these launchers take device memory only")
    if not t.is_contiguous():
        raise ValueError("tensor must be contiguous")
    if dtype is not None and t.dtype != dtype:
        raise TypeError(f"expected {dtype}, got {t.dtype}")
    return t.data_ptr()


def _f32(t):
    import torch
    return _ptr(t, torch.float32)


def _i32(t):
    import torch
    return _ptr(t, torch.int32)


# ---- launchers: same names, argument order and meaning as the reference's ----

def encoder_forward(out, inp, wte, wpe, B, T, C):
    _check(lib().encoder_forward_status(_f32(out), _i32(inp), _f32(wte), _f32(wpe), B, T, C),
           "encoder_forward")


def layernorm_forward(out, mean, rstd, inp, weight, bias, B, T, C):
    _check(lib().layernorm_forward_status(_f32(out), _f32(mean), _f32(rstd), _f32(inp),
                                          _f32(weight), _f32(bias), B, T, C), "layernorm_forward")


def fused_residual_layernorm_forward(res_out, layernorm_out, mean, rstd, inp1, inp2, weight, bias,
                                     B, T, C):
    _check(lib().fused_residual_layernorm_forward_status(
        _f32(res_out), _f32(layernorm_out), _f32(mean), _f32(rstd), _f32(inp1), _f32(inp2),
        _f32(weight), _f32(bias), B, T, C), "fused_residual_layernorm_forward")


def residual_forward(out, inp1, inp2, N):
    _check(lib().residual_forward_status(_f32(out), _f32(inp1), _f32(inp2), N), "residual_forward")


def gelu_forward(out, inp, N):
    _check(lib().gelu_forward_status(_f32(out), _f32(inp), N), "gelu_forward")


def matmul_forward(out, inp, weight, bias, B, T, C, OC):
    _check(lib().matmul_forward_status(_f32(out), _f32(inp), _f32(weight), _f32(bias), B, T, C,
                                       OC), "matmul_forward")


def matmul_forward_gelu(out, inp, weight, bias, B, T, C, OC, is_gelu):
    _check(lib().matmul_forward_gelu_status(_f32(out), _f32(inp), _f32(weight), _f32(bias), B, T,
                                            C, OC, int(bool(is_gelu))), "matmul_forward_gelu")


def matmul_forward_probe(out, inp, weight, bias, B, T, C, OC):
    """matmul_forward with the in-kernel clock probe.  Returns a (workgroups, 4) int64
    array: wall clock (10 ns ticks) at K-loop start / end, shader clock at the same."""
    import torch
    cap = ((B * T + 31) // 32) * ((OC + 31) // 32)
    probe = torch.zeros((cap, 4), dtype=torch.int64, device="cuda")
    n = ctypes.c_int(0)
    _check(lib().matmul_forward_probe_status(_f32(out), _f32(inp), _f32(weight), _f32(bias), B, T,
                                             C, OC, probe.data_ptr(), cap, ctypes.byref(n)),
           "matmul_forward_probe")
    torch.cuda.synchronize()
    return probe[:n.value].cpu().numpy()


def matmul_forward_tile_shape(B, T, C, OC):
    """(rows, columns) of the workgroup tile matmul_forward gives this problem; (0, 0) if it
    takes a kernel that is not tiled this way.  No GPU needed."""
    bm, bn = ctypes.c_int(0), ctypes.c_int(0)
    _check(lib().matmul_forward_tile_shape(B, T, C, OC, ctypes.byref(bm), ctypes.byref(bn)),
           "matmul_forward_tile_shape")
    return bm.value, bn.value


SPLITK_COUNTER_BYTES = 16384


def matmul_forward_splitk_workspace():
    """A zero-filled workspace (uint8 CUDA tensor) of the size the library recommends."""
    import torch
    return torch.zeros(lib().matmul_forward_splitk_workspace(), dtype=torch.uint8, device="cuda")


def matmul_forward_splitk(out, inp, weight, bias, B, T, C, OC, workspace, is_gelu=False, plan=None):
    """matmul_forward_gelu with a workspace that lets K be split between workgroups.
    workspace: uint8 CUDA tensor whose first SPLITK_COUNTER_BYTES were zero before its first
    use.  plan: optional (tile_rows, tile_cols, splits) to force instead of the cost model's."""
    ws, nbytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    if plan is None:
        _check(lib().matmul_forward_splitk_status(_f32(out), _f32(inp), _f32(weight), _f32(bias), B,
                                                  T, C, OC, int(bool(is_gelu)), ws, nbytes),
               "matmul_forward_splitk")
    else:
        _check(lib().matmul_forward_splitk_forced_status(_f32(out), _f32(inp), _f32(weight),
                                                         _f32(bias), B, T, C, OC, int(bool(is_gelu)),
                                                         ws, nbytes, *map(int, plan)),
               "matmul_forward_splitk_forced")


def matmul_forward_residual(out, inp, weight, bias, resid, B, T, C, OC, workspace=None):
    """out = resid + (inp . weight^T + bias), the residual add in the product's epilogue.
    workspace: as for matmul_forward_splitk (None: K is not split between workgroups)."""
    ws, nbytes = (None, 0) if workspace is None else (workspace.data_ptr(), workspace.numel())
    _check(lib().matmul_forward_residual_status(_f32(out), _f32(inp), _f32(weight), _f32(bias),
                                                _f32(resid), B, T, C, OC, ws, nbytes),
           "matmul_forward_residual")


def matmul_forward_first_columns(B, T, C, OC, workspace_bytes=0):
    """Columns computed by the first launch of a product (OC: the product is one launch)."""
    return lib().matmul_forward_first_columns(B, T, C, OC, workspace_bytes)


def forward_sums_in_matmul(config, B, T):
    """Whether gpt2_forward at this size adds the residual stream in the projections' epilogues
    (config: a dict with the GPT2Config fields, e.g. GPT2_124M).  No GPU needed."""
    cfg = GPT2Config(**config)
    return bool(lib().gpt2_forward_sums_in_matmul(ctypes.byref(cfg), B, T))


def matmul_forward_splitk_plan(B, T, C, OC, workspace_bytes):
    """(tile_rows, tile_cols, splits) that matmul_forward_splitk would use.  No GPU needed."""
    bm, bn, sp = ctypes.c_int(0), ctypes.c_int(0), ctypes.c_int(0)
    _check(lib().matmul_forward_splitk_plan(B, T, C, OC, workspace_bytes, ctypes.byref(bm),
                                            ctypes.byref(bn), ctypes.byref(sp)),
           "matmul_forward_splitk_plan")
    return bm.value, bn.value, sp.value


def attention_forward(out, qkvr, att, inp, B, T, C, NH):
    _check(lib().attention_forward_status(_f32(out), _f32(qkvr), _f32(att), _f32(inp), B, T, C,
                                          NH), "attention_forward")


_INT_MAX = 2**31 - 1  # a C int takes any whole number and drops what is above its 32 bits


class PagedCache:
    """A key/value cache in pages (GPT2PagedCache in the header).

    keys, values: contiguous CUDA tensors (num_pages, kv_heads, page_size, head_size) of float32,
    float16 or bfloat16; table: contiguous int32 CUDA tensor (B, max_pages), the pages of each
    sequence in order.  The tensors are kept alive and used in place."""

    def __init__(self, keys, values, table):
        import torch
        types = {torch.float32: 0, torch.float16: 1, torch.bfloat16: 2}  # GPT2HIP_F32, _F16, _BF16
        if keys.dtype not in types or keys.dtype != values.dtype:
            raise TypeError(f"keys and values are float32, float16 or bfloat16 alike, got {keys.dtype}, {values.dtype}")
        if keys.dim() != 4 or keys.shape != values.shape:
            raise ValueError("keys and values are (num_pages, kv_heads, page_size, head_size) alike, got "
                             f"{tuple(keys.shape)}, {tuple(values.shape)}")
        if table.dim() != 2:
            raise ValueError(f"table is (B, max_pages), got {tuple(table.shape)}")
        if max(*keys.shape, *table.shape) > _INT_MAX:
            raise ValueError(f"sizes have 32 bits, got {tuple(keys.shape)} and {tuple(table.shape)}")
        self.keys, self.values, self.table = keys, values, table
        pages, heads, size, channels = keys.shape
        self._c = GPT2PagedCache(_ptr(keys), _ptr(values), _i32(table), types[keys.dtype], pages, size,
                                 table.shape[1], heads, channels)
        self.sequences, self.kv_heads, self.head_size = table.shape[0], heads, channels
        self.page_size, self.capacity = size, size * table.shape[1]  # capacity: positions per sequence
        self._ref = ctypes.addressof(self._c)
        self._float, self._int = torch.float32, torch.int32
        self._device, self._current_device = keys.get_device(), torch.cuda.current_device
        if values.get_device() != self._device or table.get_device() != self._device:
            raise ValueError("keys, values and table are on one GPU")


def _array(t, cache, dtype, shape, what) -> int:
    """Device pointer of a contiguous tensor of that type and shape on the cache's GPU."""
    try:
        if t.dtype is dtype and t.shape == shape and t.get_device() == cache._device and t.is_contiguous():
            return t.data_ptr()
    except AttributeError:
        pass
    if not hasattr(t, "get_device") or t.get_device() != cache._device or t.dtype is not dtype:
        raise TypeError(f"{what} is a {dtype} tensor on cuda:{cache._device}, got {getattr(t, 'dtype', type(t))} on "
                        f"{getattr(t, 'device', 'the host')}")
    raise ValueError(f"{what} is contiguous and {tuple(shape)}, got {tuple(t.shape)} with strides {t.stride()}")


def _rows(inp, cache, count, floats):
    """(pointer, stride in floats) of `count` rows of at least `floats` floats; a view of a wider array will do."""
    if not hasattr(inp, "get_device") or inp.get_device() != cache._device or inp.dtype is not cache._float:
        raise TypeError(f"expected float32 rows on cuda:{cache._device}")
    shape, strides = inp.shape, inp.stride()
    if len(shape) != 2 or shape[0] < count or shape[1] < floats or (shape[1] > 1 and strides[1] != 1):
        raise ValueError(f"expected {count} rows of {floats} consecutive floats, got {tuple(shape)} with strides {strides}")
    # the stride of a single row says nothing
    stride = strides[0] if count > 1 else max(strides[0], floats)
    if stride > _INT_MAX or not 0 <= floats <= _INT_MAX or not 0 <= count <= _INT_MAX:
        raise ValueError(f"counts and strides have 32 bits, got {count} rows of {floats} floats at a stride of {stride}")
    return inp.data_ptr(), stride


def _space(workspace, cache):
    """(pointer, bytes) of a contiguous workspace on the cache's GPU."""
    if not hasattr(workspace, "get_device") or workspace.get_device() != cache._device:
        raise TypeError(f"workspace is a tensor on cuda:{cache._device}, got {getattr(workspace, 'dtype', type(workspace))} on "
                        f"{getattr(workspace, 'device', 'the host')}")
    if not workspace.is_contiguous():
        raise ValueError("workspace must be contiguous")
    return workspace.data_ptr(), workspace.nbytes


def _on_its_gpu(cache, B) -> None:
    """Launchers run on the current device: the cache has to be there, and to list B sequences."""
    if cache._current_device() != cache._device:
        raise ValueError(f"the cache is on cuda:{cache._device}, the current device is cuda:{cache._current_device()}")
    if B > cache.sequences:
        raise ValueError(f"the table lists {cache.sequences} sequences, asked for {B}")


def kv_store_paged(cache, inp, starts, lengths, N, B, NH):
    """Store the keys and values of N packed rows (q | k | v; NH = 0: k | v) into the pages: rows
    starts[b] .. starts[b + 1] - 1 become positions lengths[b] and on of sequence b."""
    _on_its_gpu(cache, B)
    rows, stride = _rows(inp, cache, N, (NH + 2 * cache.kv_heads) * cache.head_size)
    i = cache._int
    _check(lib().kv_store_paged_status(cache._ref, rows, stride, _array(starts, cache, i, (B + 1,), "starts"),
                                       _array(lengths, cache, i, (B,), "lengths"), N, B, NH), "kv_store_paged")


PAGED_COUNTER_BYTES = 65536  # GPT2HIP_PAGED_COUNTER_BYTES


def attention_decode_paged_workspace(cache, B, NH, weights=False):
    """A zero-filled workspace (uint8 CUDA tensor) that never constrains how attention_decode_paged
    splits the work.  Its first PAGED_COUNTER_BYTES stay zero between calls.  It is allocated and
    zeroed on the launchers' stream (set_stream), whatever torch's current one is: calls on that
    stream find it zero, one on another stream has to be ordered behind it."""
    import torch
    n = lib().attention_decode_paged_workspace(cache._ref, B, NH, int(weights)) if 0 < B <= _INT_MAX and 0 < NH <= _INT_MAX else 0
    if n == 0:
        raise GPT2HipError(f"attention_decode_paged_workspace: bad arguments B={B} NH={NH} kv_heads={cache.kv_heads}")
    device = cache.keys.device
    raw = lib().gpt2hip_get_stream()
    with torch.cuda.stream(torch.cuda.ExternalStream(raw, device=device) if raw else torch.cuda.default_stream(device)):
        return torch.zeros(n, dtype=torch.uint8, device=device)


def attention_decode_paged(out, cache, inp, lengths, B, NH, append=True, weights_in=None, weights_out=None,
                           workspace=None):
    """Attention of one new token per sequence over its pages.  append: inp holds packed rows and
    the new keys and values are stored as position lengths[b] first; otherwise inp holds queries
    that attend to the lengths[b] positions held.  weights_in, weights_out: accumulated attention
    weights (B, kv_heads, cache.capacity).  lengths[b] < 0: the row is left as it is."""
    _on_its_gpu(cache, B)
    f, HS = cache._float, cache.head_size
    rows, stride = _rows(inp, cache, B, (NH + 2 * cache.kv_heads if append else NH) * HS)
    win = wout = ws = None
    nbytes = 0
    if weights_in is not None:
        win = _array(weights_in, cache, f, (B, cache.kv_heads, cache.capacity), "weights_in")
    if weights_out is not None:
        wout = _array(weights_out, cache, f, (B, cache.kv_heads, cache.capacity), "weights_out")
    if workspace is not None:
        ws, nbytes = _space(workspace, cache)
    _check(lib().attention_decode_paged_status(_array(out, cache, f, (B, NH * HS), "out"), cache._ref, rows,
                                               stride, _array(lengths, cache, cache._int, (B,), "lengths"), win, wout, B, NH,
                                               1 if append else 0, ws, nbytes), "attention_decode_paged")


def kv_evict_paged(dst, src, kept, weights_out, lengths_out, weights_in, lengths, B, budget, recent):
    """Bring every sequence down to `budget` positions (the `recent` last ones and the heaviest of the
    others, each kv head for itself), copied from the pages of src into those of dst."""
    _on_its_gpu(src, B)
    _on_its_gpu(dst, B)
    if not 0 <= recent <= _INT_MAX or budget > _INT_MAX:
        raise GPT2HipError(f"kv_evict_paged: bad shape budget={budget} recent={recent}")
    f, i = src._float, src._int
    _check(lib().kv_evict_paged_status(dst._ref, src._ref, _array(kept, src, i, (B, src.kv_heads, budget), "kept"),
                                       _array(weights_out, src, f, (B, dst.kv_heads, dst.capacity), "weights_out"),
                                       _array(lengths_out, src, i, (B,), "lengths_out"),
                                       _array(weights_in, src, f, (B, src.kv_heads, src.capacity), "weights_in"),
                                       _array(lengths, src, i, (B,), "lengths"), B, budget, recent), "kv_evict_paged")


def argmax_forward(ids, logits, N, V):
    _check(lib().argmax_forward_status(_i32(ids), _f32(logits), N, V), "argmax_forward")


def matmul_forward_argmax(ids, inp, weight, bias, B, T, C, OC, workspace=None):
    """ids (B*T int32) = per-row argmax of inp . weight^T + bias, without storing the product.
    workspace: optional uint8 CUDA tensor of matmul_forward_argmax_workspace(B, T, OC) bytes."""
    import torch
    need = lib().matmul_forward_argmax_workspace(B, T, OC)
    if workspace is None:
        workspace = torch.empty(max(need, 1), dtype=torch.uint8, device="cuda")
    _check(lib().matmul_forward_argmax_status(_i32(ids), workspace.data_ptr(), workspace.numel(),
                                              _f32(inp), _f32(weight), _f32(bias), B, T, C, OC),
           "matmul_forward_argmax")


ARGMAX_NOALLOC_BYTES = 33 << 20  # GPT2HIP_ARGMAX_NOALLOC_BYTES


def matmul_forward_argmax_noalloc(ids, inp, weight, bias, B, T, C, OC):
    """matmul_forward_argmax with the pairs in the library's static device array: no
    allocation, no workspace argument; shapes beyond ARGMAX_NOALLOC_BYTES of pairs raise."""
    _check(lib().matmul_forward_argmax_noalloc_status(_i32(ids), _f32(inp), _f32(weight),
                                                      _f32(bias), B, T, C, OC),
           "matmul_forward_argmax_noalloc")


def set_stream(stream) -> None:
    """Make every launcher of this thread use `stream` (a torch.cuda.Stream, a raw
    hipStream_t value, or None for the null stream)."""
    raw = getattr(stream, "cuda_stream", stream)
    lib().gpt2hip_set_stream(raw or None)


def set_workspace(workspace) -> None:
    """Lend matmul_forward / matmul_forward_gelu of this thread a K-split workspace (a uint8
    CUDA tensor whose first SPLITK_COUNTER_BYTES were zero before its first use, e.g. from
    matmul_forward_splitk_workspace(); the caller keeps it alive), or None to take it back."""
    if workspace is None:
        _check(lib().gpt2hip_set_workspace(None, 0), "gpt2hip_set_workspace")
    else:
        _check(lib().gpt2hip_set_workspace(workspace.data_ptr(), workspace.numel()),
               "gpt2hip_set_workspace")


def read_checkpoint_config(path) -> dict:
    """Header of an llm.c checkpoint file as GPT2(**config) keywords (no GPU needed)."""
    cfg = GPT2Config()
    _check(lib().gpt2_checkpoint_read_config(os.fsencode(path), ctypes.byref(cfg)),
           "gpt2_checkpoint_read_config")
    return {name: getattr(cfg, name) for name, _ in GPT2Config._fields_}


class Timer:
    """HIP-event timer on the null stream, the stream every launcher uses."""

    def __init__(self):
        self._h = lib().gpt2hip_timer_create()
        if not self._h:
            raise GPT2HipError("gpt2hip_timer_create failed")

    def start(self):
        _check(lib().gpt2hip_timer_start(self._h), "gpt2hip_timer_start")

    def stop_ms(self) -> float:
        ms = lib().gpt2hip_timer_stop_ms(self._h)
        if ms < 0:
            raise GPT2HipError("gpt2hip_timer_stop_ms failed")
        return float(ms)

    def __del__(self):
        if getattr(self, "_h", None) and _lib is not None:  # at interpreter exit the module may be gone
            _lib.gpt2hip_timer_destroy(self._h)
            self._h = None


class GPT2:
    """The gpt2_forward driver (C++ side owns parameters and activations)."""

    def __init__(self, *, max_seq_len, vocab_size, num_layers, num_heads, channels, _handle=None):
        self.config = GPT2Config(max_seq_len, vocab_size, num_layers, num_heads, channels)
        self._h = _handle or lib().gpt2_create(ctypes.byref(self.config))
        if not self._h:
            raise GPT2HipError("gpt2_create failed: " + lib().gpt2hip_last_error().decode())
        self.num_parameters = int(lib().gpt2_num_parameters(self._h))
        self._shape = None

    @classmethod
    def from_checkpoint(cls, path):
        """Build from an llm.c fp32 checkpoint file (gpt2_124M.bin format)."""
        cfg = read_checkpoint_config(path)
        h = lib().gpt2_build_from_checkpoint(os.fsencode(path))
        if not h:
            raise GPT2HipError("gpt2_build_from_checkpoint failed: "
                               + lib().gpt2hip_last_error().decode())
        return cls(_handle=h, **cfg)

    def close(self):
        if getattr(self, "_h", None) and _lib is not None:  # at interpreter exit the module may be gone
            _lib.gpt2_destroy(self._h)
            self._h = None

    __del__ = close

    def load_params(self, host_params):
        """host_params: contiguous float32 numpy array in checkpoint order."""
        import numpy as np
        a = np.ascontiguousarray(host_params, dtype=np.float32)
        _check(lib().gpt2_load_params_host(self._h, a.ctypes.data, a.size), "gpt2_load_params_host")

    def params_tensor(self):
        """A torch view of the flat device parameter buffer (no copy)."""
        return _device_view(lib().gpt2_params_device(self._h), (self.num_parameters,), "float32")

    def reserve(self, B, T):
        _check(lib().gpt2_reserve(self._h, B, T), "gpt2_reserve")

    def forward(self, inputs):
        """inputs: (B,T) int32, numpy (host, llm.c style) or CUDA tensor (device)."""
        import numpy as np
        B, T = inputs.shape
        if isinstance(inputs, np.ndarray):
            a = np.ascontiguousarray(inputs, dtype=np.int32)
            _check(lib().gpt2_forward_status(self._h, a.ctypes.data, B, T), "gpt2_forward")
        else:
            _check(lib().gpt2_forward_device_status(self._h, _i32(inputs), B, T), "gpt2_forward")
        self._shape = (B, T)

    def prefill(self, inputs_device):
        """Run a prompt (B,T) of device ids, filling the key/value cache; returns the (B,V)
        logits of the last position (library-owned memory, overwritten by the next step)."""
        B, T = inputs_device.shape
        _check(lib().gpt2_prefill_status(self._h, _i32(inputs_device), B, T), "gpt2_prefill")
        self._step_batch = B
        return self.step_logits()

    def decode(self, next_ids_device):
        """Append one token per sequence ((B,) device ids); returns that position's (B,V) logits."""
        if next_ids_device.numel() != getattr(self, "_step_batch", -1):
            raise GPT2HipError("decode: expected one token id per prefilled sequence")
        _check(lib().gpt2_decode_status(self._h, _i32(next_ids_device)), "gpt2_decode")
        return self.step_logits()

    def generate_greedy(self, prompt_device, steps: int):
        """Greedy continuation of a (B,T) prompt of device ids by `steps` tokens: prefill, then
        argmax_forward over the step logits and one decode step per token, all queued on the
        stream with no host synchronisation in between.  Returns (B, steps) int32 device ids."""
        import torch
        B, T = prompt_device.shape
        V = self.config.vocab_size
        out = torch.empty((steps, B), dtype=torch.int32, device="cuda")
        logits = self.prefill(prompt_device)
        for s in range(steps):
            argmax_forward(out[s], logits, B, V)
            if s + 1 < steps:
                logits = self.decode(out[s])
        self.decode_sync()  # a step that failed on the device would have left NaN logits behind
        return out.t().contiguous()

    def decode_sync(self) -> None:
        """Wait for the decode steps queued so far; raises if one of them gave up on the device
        (the cache is then rolled back to the positions before it, see cache_length())."""
        _check(lib().gpt2_decode_sync_status(self._h), "gpt2_decode_sync")

    def decode_probe(self, next_ids_device):
        """One decode step of the persistent kernel with its clock probe: returns a
        (phases, 2, workgroups) int64 tensor of 100 MHz wall-clock readings (work done / barrier
        passed) -- see gpt2_decode_probe_status in the header."""
        import torch
        n = lib().gpt2_decode_probe_size(self._h)
        if n == 0:
            raise GPT2HipError("decode_probe: the persistent kernel does not take this model")
        clocks = torch.zeros(n, dtype=torch.int64, device="cuda")
        _check(lib().gpt2_decode_probe_status(self._h, _i32(next_ids_device), clocks.data_ptr(), n),
               "gpt2_decode_probe")
        phases = 5 * self.config.num_layers + 1
        return clocks.view(phases, 2, -1)

    def decode_probe_size(self) -> int:
        """Clock slots decode_probe needs; 0 if the next step would not be the persistent kernel."""
        return int(lib().gpt2_decode_probe_size(self._h))

    def decode_options(self, persistent: bool = True, spin_limit: int = 1 << 21):
        """Choose between the persistent decode-step kernel and one launch per operation."""
        _check(lib().gpt2_decode_options(self._h, int(persistent), spin_limit), "gpt2_decode_options")

    def step_logits(self):
        return _device_view(lib().gpt2_step_logits(self._h),
                            (self._step_batch, self.config.vocab_size), "float32")

    def cache_length(self) -> int:
        return lib().gpt2_cache_length(self._h)

    def forward_graph(self, inputs_device):
        """forward() of device ids, replayed from a HIP graph captured on first use per (B,T)."""
        B, T = inputs_device.shape
        _check(lib().gpt2_forward_graph_status(self._h, _i32(inputs_device), B, T),
               "gpt2_forward_graph")
        self._shape = (B, T)

    def forward_argmax(self, inputs_device):
        """Forward that keeps only each position's argmax token id; returns (B,T) int32."""
        import torch
        B, T = inputs_device.shape
        ids = torch.empty((B, T), dtype=torch.int32, device="cuda")
        _check(lib().gpt2_forward_argmax_status(self._h, _i32(inputs_device), B, T,
                                                ids.data_ptr()), "gpt2_forward_argmax")
        self._shape = (B, T)
        return ids

    def forward_profiled(self, inputs_device):
        """Forward with per-launch HIP events; returns {category: ms} for this pass."""
        B, T = inputs_device.shape
        ms = (ctypes.c_float * len(PROF_CATEGORIES))()
        _check(lib().gpt2_forward_profiled_status(self._h, _i32(inputs_device), B, T, ms),
               "gpt2_forward_profiled")
        self._shape = (B, T)
        return dict(zip(PROF_CATEGORIES, (float(x) for x in ms)))

    def logits(self):
        B, T = self._shape
        return _device_view(lib().gpt2_logits(self._h), (B, T, self.config.vocab_size), "float32")

    def lnf(self):
        B, T = self._shape
        return _device_view(lib().gpt2_lnf(self._h), (B, T, self.config.channels), "float32")

    def argmax(self):
        import torch
        B, T = self._shape
        ids = torch.empty((B, T), dtype=torch.int32, device="cuda")
        _check(lib().gpt2_argmax_status(self._h, ids.data_ptr()), "gpt2_argmax")
        return ids


def _device_view(ptr: int, shape, dtype: str):
    """Wrap library-owned device memory as a torch tensor without copying."""
    import numpy as np
    import torch

    class _Holder:
        pass

    h = _Holder()
    n = int(np.prod(shape))
    h.__cuda_array_interface__ = {
        "shape": (n,), "typestr": {"float32": "<f4", "int32": "<i4"}[dtype],
        "data": (int(ptr), False), "version": 3, "strides": None,
    }
    return torch.as_tensor(h, device="cuda").view(*shape)
