"""ctypes binding of ``libhf_convrot.so`` and ``libhf_block.so`` (the C ABIs of include/hf_convrot.h, and of
include/hf_block.h and include/hf_cache.h) and the build recipe that makes them.

Each library is built in-tree by ``build_library()`` (hipcc, gfx950) and loaded from next to this file. There is no
fallback: when one is missing or does not load, ``library()`` or ``block_library()`` raises.
"""

from __future__ import annotations

import ctypes
import os
import struct
import subprocess
from concurrent.futures import ThreadPoolExecutor
from functools import lru_cache

PACKAGE_DIR = os.path.dirname(os.path.abspath(__file__))
REPO_DIR = os.path.dirname(PACKAGE_DIR)
LIB_PATH = os.path.join(PACKAGE_DIR, "libhf_convrot.so")
SOURCE = os.path.join(PACKAGE_DIR, "csrc", "convrot_abi.hip")
#: The operators around the INT8 linears of a block (include/hf_block.h, include/hf_cache.h), a library of their own.
BLOCK_LIB_PATH = os.path.join(PACKAGE_DIR, "libhf_block.so")
BLOCK_SOURCE = os.path.join(PACKAGE_DIR, "csrc", "block_abi.hip")
#: The benchmark's calibration kernels (matrix-core ceiling), a library of their own outside the C ABI.
CEILINGS_LIB_PATH = os.path.join(PACKAGE_DIR, "libhf_ceilings.so")
CEILINGS_SOURCE = os.path.join(PACKAGE_DIR, "csrc", "ceilings.hip")
ARCH = "gfx950"

#: hipcc flags: CDNA4 only; fp-contract off keeps every multiply and add separately rounded as written; packed
#: fp32 instructions are disabled.
HIPCC_FLAGS = [
    f"--offload-arch={ARCH}",
    "-O3",
    "-std=c++17",
    "-fPIC",
    "-shared",
    "-ffp-contract=off",
    "-Xclang", "-target-feature", "-Xclang", "-packed-fp32-ops",
]

HF_OK = 0
STATUS_NAMES = {
    -1: "HF_ERR_ARGUMENT",
    -2: "HF_ERR_GROUP",
    -3: "HF_ERR_ALIGNMENT",
    -4: "HF_ERR_LAUNCH",
    -5: "HF_ERR_SIZE",
    -6: "HF_ERR_SCRATCH",
}

#: Every function include/hf_convrot.h declares, with its ctypes signature.
_P, _I64, _I32 = ctypes.c_void_p, ctypes.c_int64, ctypes.c_int32
SIGNATURES = {
    "hf_version": ([], ctypes.c_char_p),
    "hf_strerror": ([ctypes.c_int], ctypes.c_char_p),
    "hf_rotate_quant": ([_P, _I64, _P, _I64, _P, _I64, _I64, _I32, _P], ctypes.c_int),
    "hf_rotate_quant_ex": ([_P, _I64, _P, _I64, _P, _I64, _I64, _I32, _I32, _P], ctypes.c_int),
    "hf_lowrank_down": ([_P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I32, _P], ctypes.c_int),
    "hf_lowrank_down_ws_bytes": ([_I64, _I64, _I32], ctypes.c_int64),
    "hf_lowrank_down_ws": ([_P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I32, _P, _I64, _P], ctypes.c_int),
    "hf_int8_linear_ws_bytes": ([_I64, _I64, _I64, _I32, _I32], ctypes.c_int64),
    "hf_int8_linear_ws": ([_P, _I64, _P, _I64, _P, _P, _P, _I64, _P, _I64, _I32, _P, _P, _I64, _I64, _I64, _I64, _P,
                           _I64, _P], ctypes.c_int),
    "hf_int8_linear_act_ws": ([_P, _I64, _P, _I64, _P, _P, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _I64, _I64, _I64,
                               _I64, _P, _I64, _P], ctypes.c_int),
    "hf_lowrank_up": ([_P, _I64, _P, _I64, _I32, _P, _P, _I64, _I64, _I64, _P], ctypes.c_int),
    "hf_int8_linear": ([_P, _I64, _P, _I64, _P, _P, _P, _I64, _P, _I64, _I32, _P, _P, _I64, _I64, _I64, _I64, _P],
                       ctypes.c_int),
    "hf_int8_gemm_i32": ([_P, _I64, _P, _I64, _P, _I64, _I64, _I64, _I64, _P], ctypes.c_int),
    "hf_convrot_linear_ws_bytes": ([_I64, _I64, _I64, _I32, _I32], ctypes.c_int64),
    "hf_convrot_linear_ws": ([_P, _I64, _P, _P, _I32, _I32, _P, _I64, _P, _P, _I64, _P, _I64, _I32, _P, _I32, _I32,
                              _P, _P, _I64, _I64, _I64, _I64, _P, _I64, _P], ctypes.c_int),
    "hf_convrot_linear": ([_P, _I64, _P, _I64, _P, _P, _I64, _P, _I64, _I32, _P, _I32, _P, _P, _P, _P, _I64, _I64,
                           _I64, _I64, _P], ctypes.c_int),
    "hf_route": ([_I32, _I64, _I64, _I64, _I32], ctypes.c_int32),
    "hf_convrot_linear_noalloc_max_bytes": ([], ctypes.c_int64),
    "hf_convrot_linear_noalloc": ([_P, _I64, _P, _P, _I32, _I32, _P, _I64, _P, _P, _I64, _P, _I64, _I32, _P, _I32,
                                   _I32, _P, _P, _I64, _I64, _I64, _I64, _P], ctypes.c_int),
}

#: Every function include/hf_block.h declares.
_F = ctypes.c_float
BLOCK_SIGNATURES = {
    "hf_qk_norm_rope": ([_P, _I64, _I64, _I32, _P, _I64, _I64, _I32, _P, _I64, _I64, _P, _I64, _I64, _P, _I32, _I64,
                         _I32, _P, _P, _I32, _I32, _I32, _P, _P, _I32, _F, _I64, _I32, _I32, _P], ctypes.c_int),
    "hf_attention_plan": ([_P, _P, _I64, _I32, _I32, _I32, _I32, _I32, _P, _I64], ctypes.c_int64),
    "hf_attention_ws_bytes": ([_P, _I64], ctypes.c_int64),
    "hf_attention": ([_P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _P, _I64, _I64, _F, _P, _P, _I64, _P, _I64,
                      _I32, _P], ctypes.c_int),
    "hf_adapter_plan": ([_P, _P, _I64, _I32, _I32, _P, _I64], ctypes.c_int64),
    "hf_adapter_ws_bytes": ([_P, _I64, _I64, _I32, _I32], ctypes.c_int64),
    "hf_adapter_add": ([_P, _I64, _P, _I64, _P, _P, _I32, _P, _P, _I64, _I64, _I64, _P, _P, _I64, _P, _I64, _I32, _P],
                       ctypes.c_int),
    "hf_qk_norm_rope_call": ([ctypes.c_char_p], ctypes.c_int),
    "hf_attention_call": ([ctypes.c_char_p], ctypes.c_int),
    "hf_adapter_add_call": ([ctypes.c_char_p], ctypes.c_int),
}

#: Every function include/hf_cache.h declares (of the same library as hf_block.h's).
CACHE_SIGNATURES = {
    "hf_cache_page_bytes": ([_I32, _I32, _I32], ctypes.c_int64),
    "hf_cache_plan": ([_P, _P, _P, _I64, _P, _I64, _I32, _I32, _I32, _I32, _I32, _I32, _P, _I64], ctypes.c_int64),
    "hf_cache_ws_bytes": ([_P, _I64], ctypes.c_int64),
    "hf_cache_append": ([ctypes.c_char_p], ctypes.c_int),
    "hf_cache_read": ([ctypes.c_char_p], ctypes.c_int),
    "hf_cached_attention": ([ctypes.c_char_p], ctypes.c_int),
    "hf_copy_pages": ([ctypes.c_char_p], ctypes.c_int),
    "hf_residual_norm": ([ctypes.c_char_p], ctypes.c_int),
}

#: The launches' parameters as the structs of hf_block.h and hf_cache.h lay them out.
ROPE_ARGS = struct.Struct("@PqqiPqqiPqqPqqPiqiPPiiiPPifqiiP")
ATTENTION_ARGS = struct.Struct("@PqqPqqPqqPqqfPPqPqiP")
ADAPTER_ARGS = struct.Struct("@PqPqPPiPPqqqPPqPqiP")
CACHE_APPEND_ARGS = struct.Struct("@PqqPqqPPPqiP")
CACHE_READ_ARGS = struct.Struct("@PPPPPqiP")
CACHED_ATTENTION_ARGS = struct.Struct("@PqqPPqqfPPqPqiP")
COPY_PAGES_ARGS = struct.Struct("@PqqqqPPqP")
RESIDUAL_NORM_ARGS = struct.Struct("@PqPqPqPqPqPqPqPPPqqiiiiiiiffP")

#: Queries of hf_route.
ROUTE_UP_ROWS, ROUTE_ROTATE_LOWRANK, ROUTE_STREAM_WEIGHT = 0, 1, 2


def hipcc() -> str:
    rocm = os.environ.get("ROCM_PATH", "/opt/rocm")
    path = os.path.join(rocm, "bin", "hipcc")
    return path if os.path.exists(path) else "hipcc"


def _compile(source: str, target: str, verbose: bool) -> None:
    tmp = target + ".tmp"
    proc = subprocess.run([hipcc(), *HIPCC_FLAGS, "-o", tmp, source], capture_output=True, text=True)
    if proc.returncode != 0:
        raise RuntimeError(f"hipcc failed ({proc.returncode}) on {source}:\n{proc.stderr[-4000:]}")
    if verbose and proc.stderr:
        print(proc.stderr[-2000:])
    os.replace(tmp, target)


def build_library(verbose: bool = False) -> str:
    """Compile csrc/ into libhf_convrot.so, libhf_block.so and the benchmark's libhf_ceilings.so, for gfx950 (always
    recompiles), side by side. Returns the convrot library's path."""
    with ThreadPoolExecutor(3) as pool:
        jobs = [pool.submit(_compile, source, target, verbose) for source, target in
                ((SOURCE, LIB_PATH), (BLOCK_SOURCE, BLOCK_LIB_PATH), (CEILINGS_SOURCE, CEILINGS_LIB_PATH))]
    for job in jobs:
        job.result()
    library.cache_clear()
    block_library.cache_clear()
    ceilings_library.cache_clear()
    return LIB_PATH


def _load(path: str, signatures: dict) -> ctypes.CDLL:
    if not os.path.exists(path):
        raise RuntimeError(
            f"{path} is missing: build it with `python -c 'import __graft_entry__ as g; g.build()'` "
            "(hipcc --offload-arch=gfx950)"
        )
    try:
        lib = ctypes.CDLL(path)
    except OSError as exc:
        raise RuntimeError(f"cannot load {path}: {exc}") from exc
    for name, (argtypes, restype) in signatures.items():
        fn = getattr(lib, name)
        fn.argtypes = argtypes
        fn.restype = restype
    return lib


@lru_cache(maxsize=None)
def library() -> ctypes.CDLL:
    """The loaded library with argument types set. Raises RuntimeError when it is missing or does not load."""
    return _load(LIB_PATH, SIGNATURES)


@lru_cache(maxsize=None)
def block_library() -> ctypes.CDLL:
    """The attention block's operators, as `library`."""
    return _load(BLOCK_LIB_PATH, {**BLOCK_SIGNATURES, **CACHE_SIGNATURES})


@lru_cache(maxsize=None)
def ceilings_library() -> ctypes.CDLL:
    """The benchmark's calibration library (csrc/ceilings.hip). Raises RuntimeError when it is missing."""
    if not os.path.exists(CEILINGS_LIB_PATH):
        raise RuntimeError(f"{CEILINGS_LIB_PATH} is missing: build it with `python -c 'import __graft_entry__ as g; "
                           "g.build()'`")
    lib = ctypes.CDLL(CEILINGS_LIB_PATH)
    lib.hf_ceiling_mfma_i8.argtypes = [_P, _I32, _I32, _P, _P]
    lib.hf_ceiling_mfma_i8.restype = ctypes.c_int
    lib.hf_ceiling_mfma_i8_macs.argtypes = [_I32, _I32]
    lib.hf_ceiling_mfma_i8_macs.restype = ctypes.c_int64
    lib.hf_ceiling_stream.argtypes = [_P, _P, _I64, _I32, _I32, _I32, _I32, _P, _P]
    lib.hf_ceiling_stream.restype = ctypes.c_int
    return lib


def status_text(status: int) -> str:
    return f"{STATUS_NAMES.get(status, status)}: {library().hf_strerror(status).decode()}"
