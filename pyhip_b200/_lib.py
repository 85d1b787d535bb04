"""ctypes binding of libb200moe.so (the C ABI declared in include/b200moe.h).

Mirrors how the reference reaches its kernels: a lazily loaded, cached ``ctypes.CDLL`` handle,
raw device pointers and the current torch stream passed as ``void*``
(src/core/hiptools.py:10-35,82-100 of tingqli/pyhip); a non-zero status becomes a Python
exception, as the reference's ``HIP error`` exceptions do (hiptools.py:37-39).

The dense operators around the layer (`dense()`) are reached through a torch binding that calls the same C ABI.

There is no fallback: if the shared library is missing or fails to load, importing callers
get an ImportError / RuntimeError that says how to build it.
"""
from __future__ import annotations

import ctypes
import functools
import pathlib
import shutil
import subprocess

PKG_DIR = pathlib.Path(__file__).resolve().parent
CSRC = PKG_DIR / "csrc"
LIB_PATH = PKG_DIR / "libb200moe.so"
DENSE_PATH = PKG_DIR / "_dense.so"          # torch binding of the dense operators (csrc/dense_torch.cpp)
SOURCES = ["api.cu", "moe_aux.cu", "moe_gemm_sm100.cu", "moe_gemm_fp8_sm100.cu", "moe_gemm_bf16_sm100.cu",
           "moe_batch1.cu", "forward_static.cu", "block_norm.cu", "router_train.cu", "linear_int8_sm100.cu"]
NVCC_FLAGS = ["-gencode", "arch=compute_100a,code=sm_100a", "-lineinfo", "-O3", "-std=c++17",
              "--threads", "0", "-shared", "-Xcompiler", "-fPIC"]

W_MXFP4, W_FP8_128, W_FP8_ROW, W_BF16 = 0, 1, 2, 3
ACT_SILU, ACT_SWIGLU = 0, 1
COMBINE_GATHER, COMBINE_FUSED = 0, 1
ACTQ_TERMS, ACTQ_1X128 = 0, 1
ABI_VERSION = 3
T_BF16, T_FP16, T_FP32, T_INT8 = 0, 1, 2, 3
LINEAR_HOLD_BACK = 256
GATE_NONE, GATE_CHANNEL, GATE_TOKEN, GATE_FULL = 0, 1, 2, 3


class Shape(ctypes.Structure):
    _fields_ = [("T", ctypes.c_int32), ("K", ctypes.c_int32), ("E", ctypes.c_int32),
                ("E_route", ctypes.c_int32), ("H", ctypes.c_int32), ("I", ctypes.c_int32),
                ("B", ctypes.c_int32), ("weight_format", ctypes.c_int32),
                ("activation", ctypes.c_int32), ("swiglu_limit", ctypes.c_float),
                ("act_terms", ctypes.c_int32), ("combine_mode", ctypes.c_int32),
                ("act_quant", ctypes.c_int32), ("doweight_stage1", ctypes.c_int32), ("cta_pairs", ctypes.c_int32)]


_WS_FIELDS = ["total_bytes", "max_rows", "off_sorted_ids", "off_sorted_w", "off_sorted_e",
              "off_num_valid", "off_loc", "off_status", "off_xq", "off_xsf", "off_hq", "off_hsf", "off_out2",
              "off_sort_scratch"]


class Workspace(ctypes.Structure):
    _fields_ = [(n, ctypes.c_int64) for n in _WS_FIELDS]


class Io(ctypes.Structure):
    """b200moe_io: every tensor of one layer call (optional ones may be None)."""
    _fields_ = [(n, ctypes.c_void_p) for n in ("x_bf16", "topk_ids", "topk_weight", "expert_mask", "num_local_tokens",
                                               "w1_q", "w1_scale_prepared", "w2_q", "w2_scale_prepared", "bias1",
                                               "bias2", "y_bf16")]


EXPORTS = ["b200moe_version", "b200moe_last_error", "b200moe_workspace_layout",
           "b200moe_prepared_scale_bytes", "b200moe_prepare_scales", "b200moe_sort_align",
           "b200moe_quant_rows", "b200moe_quant_rows_e4m3", "b200moe_gateup", "b200moe_down", "b200moe_combine",
           "b200moe_forward", "b200moe_forward_dyn", "b200moe_sort_align_dyn", "b200moe_sort_align_ws",
           "b200moe_sort_scratch_bytes", "b200moe_route_topk", "b200moe_forward_static", "b200moe_gather_sum", "b200moe_debug_probe",
           "b200moe_forward_ex", "b200moe_static_status", "b200moe_ep_plan", "b200moe_quant_rows_fp8_1x128",
           "b200moe_forward_batch1", "b200moe_batch1_scratch_bytes",
           "b200moe_quantize_int8", "b200moe_linear_int8", "b200moe_linear_int8_workspace", "b200moe_linear_int8_status", "b200moe_block_norm", "b200moe_block_norm_bwd",
           "b200moe_block_norm_bwd_workspace", "b200moe_router_workspace", "b200moe_router_forward",
           "b200moe_router_backward"]


def _stale(target, deps) -> bool:
    return not target.exists() or any(target.stat().st_mtime < d.stat().st_mtime for d in deps)


def _dense_tag() -> str:
    """What the torch binding is built against; it stands in the file as text."""
    import sys

    import torch
    return f"dense binding for torch {torch.__version__}, {sys.implementation.cache_tag}"


def _dense_fits() -> bool:
    return DENSE_PATH.exists() and f"{_dense_tag()}\0".encode() in DENSE_PATH.read_bytes()


def _dense_command():
    import sysconfig

    import torch
    root = pathlib.Path(torch.__file__).resolve().parent
    cuda = pathlib.Path(shutil.which("nvcc") or "/usr/local/cuda/bin/nvcc").resolve().parents[1]
    inc = [root / "include", root / "include/torch/csrc/api/include", sysconfig.get_paths()["include"], cuda / "include"]
    return ["g++", "-O2", "-std=c++17", "-shared", "-fPIC", "-fvisibility=hidden", "-DTORCH_EXTENSION_NAME=_dense",
            "-DTORCH_API_INCLUDE_EXTENSION_H", f'-DB200MOE_DENSE_TAG="{_dense_tag()}"', f"-D_GLIBCXX_USE_CXX11_ABI={int(torch._C._GLIBCXX_USE_CXX11_ABI)}",
            *(f"-isystem{i}" for i in inc), "-o", str(DENSE_PATH), str(CSRC / "dense_torch.cpp"), f"-L{root / 'lib'}", "-lc10",
            "-lc10_cuda", "-ltorch", "-ltorch_cpu", "-ltorch_python", f"-L{PKG_DIR}", "-l:libb200moe.so", "-Wl,-rpath,$ORIGIN",
            f"-Wl,-rpath,{root / 'lib'}"]


def build(force: bool = False, verbose: bool = False) -> pathlib.Path:
    """Compile the CUDA sources for sm_100a into pyhip_b200/libb200moe.so (nvcc cross-compiles
    without a GPU) and the torch binding of the dense operators into pyhip_b200/_dense.so."""
    header = PKG_DIR.parent / "include" / "b200moe.h"
    srcs = [CSRC / s for s in SOURCES]
    if force or _stale(LIB_PATH, srcs + list(CSRC.glob("*.h")) + list(CSRC.glob("*.cuh")) + [header]):
        cmd = ["nvcc", *NVCC_FLAGS, "-o", str(LIB_PATH), *map(str, srcs)]
        if verbose:
            cmd.insert(1, "-Xptxas=-v")
        res = subprocess.run(cmd, capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("nvcc failed:\n" + res.stdout + res.stderr)
        if verbose:
            print(res.stderr)
    if force or _stale(DENSE_PATH, [CSRC / "dense_torch.cpp", header]) or not _dense_fits():
        res = subprocess.run(_dense_command(), capture_output=True, text=True)
        if res.returncode != 0:
            raise RuntimeError("g++ failed:\n" + res.stdout + res.stderr)
    return LIB_PATH


@functools.cache
def lib() -> ctypes.CDLL:
    if not LIB_PATH.exists():
        raise ImportError(f"{LIB_PATH} is missing: run `python -c 'import __graft_entry__ as g; g.build()'` "
                          "(needs nvcc); this package has no CPU or eager fallback")
    L = ctypes.CDLL(str(LIB_PATH))
    # before anything else is bound: a library of another version need not have the entries, nor these arguments
    L.b200moe_version.restype = ctypes.c_int
    missing = [n for n in EXPORTS if not hasattr(L, n)]
    if missing or L.b200moe_version() != ABI_VERSION:
        raise RuntimeError(f"libb200moe.so version mismatch; rebuild it (version {L.b200moe_version()} of {ABI_VERSION}, "
                           f"missing: {', '.join(missing) or 'nothing'})")
    vp, i32, i64 = ctypes.c_void_p, ctypes.c_int32, ctypes.c_int64
    sp, wp = ctypes.POINTER(Shape), ctypes.POINTER(Workspace)
    L.b200moe_last_error.restype = ctypes.c_char_p
    L.b200moe_workspace_layout.argtypes = [sp, wp]
    L.b200moe_prepared_scale_bytes.argtypes = [sp, ctypes.c_int, ctypes.POINTER(i64)]
    L.b200moe_prepare_scales.argtypes = [sp, ctypes.c_int, vp, vp, vp]
    L.b200moe_sort_align.argtypes = [vp, vp, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp]
    L.b200moe_quant_rows.argtypes = [vp, i32, vp, vp, i32, i32, i32, i32, i32, i64, vp, vp, vp]
    L.b200moe_quant_rows_e4m3.argtypes = [vp, i32, vp, vp, i32, i32, i32, i32, i64, vp, vp, vp]
    L.b200moe_quant_rows_fp8_1x128.argtypes = [vp, i32, vp, vp, i32, i32, i32, i32, i64, vp, vp, vp]
    L.b200moe_gateup.argtypes = [sp, wp, vp, vp, vp, vp, vp, vp]
    L.b200moe_down.argtypes = [sp, wp, vp, vp, vp, vp, vp, vp]
    L.b200moe_forward_ex.argtypes = [sp, wp, vp, ctypes.POINTER(Io), vp]
    L.b200moe_static_status.argtypes = [sp, vp, vp]
    L.b200moe_combine.argtypes = [sp, wp, vp, vp, vp, vp]
    L.b200moe_forward.argtypes = [sp, wp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp]
    L.b200moe_forward_dyn.argtypes = [sp, wp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp]
    L.b200moe_sort_align_dyn.argtypes = [vp, vp, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp]
    L.b200moe_sort_align_ws.argtypes = [vp, vp, i32, i32, i32, i32, vp, vp, vp, vp, vp, vp, vp, vp, i64, vp]
    L.b200moe_sort_scratch_bytes.argtypes = [i32, ctypes.POINTER(i64)]
    L.b200moe_route_topk.argtypes = [vp, i32, i32, i32, i32, i32, vp, vp, vp]
    L.b200moe_forward_static.argtypes = [sp, vp, vp, vp, vp, vp, vp, vp, vp, vp, vp]
    L.b200moe_forward_batch1.argtypes = [sp] + [vp] * 14
    L.b200moe_batch1_scratch_bytes.argtypes = [sp, ctypes.POINTER(ctypes.c_int64)]
    L.b200moe_gather_sum.argtypes = [vp, vp, i32, i32, i32, vp, vp]
    L.b200moe_ep_plan.argtypes = [vp, i32, i32, i32, i32, vp, vp, vp, vp]
    L.b200moe_debug_probe.argtypes = [ctypes.c_int, vp, vp, vp]
    f32 = ctypes.c_float
    norm = [vp, i64, vp, i64, vp, vp, i64, vp, i32, i32, i32, i32, i32, f32]
    L.b200moe_quantize_int8.argtypes = [vp, i64, i32, i32, i32, vp, vp, vp]
    L.b200moe_linear_int8.argtypes = [vp, i64, i32, vp, vp, vp, vp, i32, i32, i32, i32, i32, vp, i64, vp, vp, vp]
    L.b200moe_linear_int8_workspace.argtypes = [i32, i32, i32, i32, ctypes.POINTER(i64)]
    L.b200moe_linear_int8_status.argtypes = [ctypes.POINTER(i32)]
    L.b200moe_block_norm.argtypes = norm + [f32] + [vp] * 6
    L.b200moe_block_norm_bwd.argtypes = norm + [vp] * 8 + [vp, i64, vp]
    L.b200moe_block_norm_bwd_workspace.argtypes = [i32, i32, i32, ctypes.POINTER(i64)]
    L.b200moe_router_workspace.argtypes = [i32, i32, i32, ctypes.POINTER(i64)]
    L.b200moe_router_forward.argtypes = [vp, i64] + [i32] * 6 + [vp, vp, i32] + [vp] * 10 + [i64, vp]
    L.b200moe_router_backward.argtypes = [vp, i64] + [i32] * 6 + [vp] * 11
    for name in EXPORTS:
        if name not in ("b200moe_version", "b200moe_last_error"):
            getattr(L, name).restype = ctypes.c_int
    return L


class B200MoEError(RuntimeError):
    pass


@functools.cache
def dense():
    """The torch binding of the dense operators.  Like `lib()` it has no fallback."""
    lib()                                   # the library that it links against, of the version that it was built for
    if not DENSE_PATH.exists():
        raise ImportError(f"{DENSE_PATH} is missing: run `python -c 'import __graft_entry__ as g; g.build()'`")
    if not _dense_fits():                   # loading it could end the process
        raise ImportError(f"{DENSE_PATH} was built for another torch or Python than this one ({_dense_tag()}): rebuild it")
    import importlib.util

    import torch  # noqa: F401  (its libraries have to be loaded first)
    spec = importlib.util.spec_from_file_location("pyhip_b200._dense", DENSE_PATH)
    module = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(module)
    module.set_error(B200MoEError)
    return module


def check(rc: int, what: str) -> None:
    if rc != 0:
        msg = lib().b200moe_last_error().decode(errors="replace")
        kind = "argument error" if rc < 0 else f"CUDA error {rc}"
        raise B200MoEError(f"{what}: {kind}: {msg}")


def workspace_layout(shape: Shape) -> Workspace:
    ws = Workspace()
    check(lib().b200moe_workspace_layout(ctypes.byref(shape), ctypes.byref(ws)), "workspace_layout")
    return ws
