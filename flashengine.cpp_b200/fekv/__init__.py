"""fekv — host-side binding of the B200 paged-KV hot path.

* :mod:`fekv._lib`      ctypes binding of ``include/fe_kv.h``
  (``lib/libfe_kv_b200.so``; no fallback when it is missing).
* :mod:`fekv.ops`       the reference's ``fe::cuda`` operator interface
  (``create_plan``/``prepare_plan``/``attention``/``store``/``rope``/
  ``accept``) plus the fused ``rope_append`` and block copy, and the
  8-bit cache (``Kv8Pool``, ``append_kv8``, ``Kv8Plan``, ``gather_kv8``,
  ``copy_blocks_kv8``).
* :mod:`fekv.metadata`  the per-step slot mapping / page tables of
  ``CudaModel::prepare``.
* :mod:`fekv.workloads` seeded synthetic configs C1..C5.
"""
from . import metadata, workloads  # noqa: F401
from ._lib import (FE_DTYPE_BF16, FE_DTYPE_F16, FE_KV8_BLOCK as KV8_BLOCK,  # noqa: F401
                   FeError, LIB_PATH, SHIM_PATH, load)
from .ops import (AttentionPlan, HostKv8Plan, HostPlan, Kv8Plan, Kv8Pool,  # noqa: F401
                  accept, append_kv8, attention, clear_pages, copy_blocks,
                  copy_blocks_kv8, create_plan, destroy_plan, device_errors, fork_copies, gather, gather_kv8,
                  paged_decode_noalloc, prepare_plan, rope, rope_append, store)
