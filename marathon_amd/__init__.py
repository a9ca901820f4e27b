"""marathon_amd: the shift-connector KV reuse path of acrosley/marathon on MI355X.

Host API (mirrors src/marathon/shift_kernels.py and src/marathon/shift_store.py):
``rope_shift``, ``RopeShift``, ``scatter_shifted``, ``use_hip``, ``warmup``,
``ShiftStore``, ``SessionTable``, ``slots``, ``plan_load``, ``plan_save``; the
block-layout :class:`BlockShiftStore` (preallocated pool, per-position validity); batched
launches through :class:`marathon_amd.spans.ShiftPlan`; the worker-side load path in
:mod:`marathon_amd.connector`.  The same for a cache held in 8 bits with a scale for each
block of tokens and head (:mod:`marathon_amd.scaled_cache`): :class:`ScaledCache`, its step's
tables and slots (:func:`step_slots`), :func:`store_scaled`, :func:`attend_scaled` and
:class:`ScaledShifts`.  Everything that touches KV runs in hand-written gfx950 kernels
(``csrc/*.hip``) behind the C ABI in ``include/``.
"""

from .block_store import BlockShiftStore
from .scaled_cache import (
    ScaledCache,
    ScaledShifts,
    StepSlots,
    attend_scaled,
    step_slots,
    store_scaled,
)
from .shift_kernels import RopeShift, inv_freq_for, rope_shift, scatter_shifted, use_hip, warmup
from .shift_store import (
    DEFAULT_STORE_TOKENS,
    SLAB,
    LoadDecision,
    SessionTable,
    ShiftStore,
    plan_load,
    plan_save,
    slots,
)

__all__ = [
    "RopeShift",
    "inv_freq_for",
    "rope_shift",
    "scatter_shifted",
    "use_hip",
    "warmup",
    "DEFAULT_STORE_TOKENS",
    "SLAB",
    "LoadDecision",
    "SessionTable",
    "ShiftStore",
    "BlockShiftStore",
    "plan_load",
    "plan_save",
    "slots",
    "ScaledCache",
    "ScaledShifts",
    "StepSlots",
    "attend_scaled",
    "step_slots",
    "store_scaled",
]
