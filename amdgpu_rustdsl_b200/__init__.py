"""B200 (sm_100a) implementation of the reference's MXFP8 attention forward path `fmha_fwd_hd128_mxfp8_auto`.

`fmha_fwd_mxfp8` / `select_path` mirror python/amdgpu_jit/ops.py of the reference; `_abi` binds the C ABI of
include/fmha_mxfp8_abi.h. The CUDA library is built in-tree (csrc/Makefile); there is no other backend.
"""
from ._abi import ContractError  # noqa: F401
from .kv4 import Kv4Cache, fmha_fwd_kv4, kv4_append, kv4_evict, kv4_pool, kv4_read  # noqa: F401
from .kv8 import Kv8Cache, fmha_fwd_kv8, kv8_append, kv8_pool, kv8_read  # noqa: F401
from .ops import Q_PRESCALE, device_status, fmha_fwd_mxfp8, quantize_qk, quantize_v, reset_workspaces, select_path  # noqa: F401
from .pages import pages_cut, pages_stack, pages_take  # noqa: F401
from .rope import Rope, rope_frequencies, rope_rotate  # noqa: F401
