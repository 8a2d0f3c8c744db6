"""``ops_rec.ascendc.attention`` -- attribute access is forwarded to ``torch.ops.ops_rec``.

Same surface as the reference module (ops_rec/ascendc/attention/__init__.py:31-55): both
``ops_rec.ascendc.attention.hstu_jagged(...)`` and ``from ops_rec.ascendc.attention import
hstu_jagged`` work, and an unknown name raises ``AttributeError`` listing what exists.  The ``hstu_paged_fp8*`` operators (an 8-bit paged cache)
and ``rotary`` (positions on queries and keys) are extensions: the reference has none of the kind.
"""

import torch

_NS = torch.ops.ops_rec
_OPS = ("hstu_jagged", "hstu_jagged_backward", "hstu_dense", "hstu_dense_backward", "hstu_paged",
        "hstu_paged_fp8", "hstu_paged_fp8_append", "hstu_paged_fp8_evict", "rotary")  # fmt: skip

__all__ = [name for name in _OPS if hasattr(_NS, name)]
for _name in __all__:
    globals()[_name] = getattr(_NS, _name)


def __getattr__(name: str):
    if not name.startswith("_") and hasattr(_NS, name):
        return getattr(_NS, name)
    raise AttributeError(
        f"module '{__name__}' has no attribute '{name}'. Operator '{name}' is not built for gfx950. "
        f"Available ops: {sorted(__all__)}"
    )


def __dir__():
    return sorted(set(globals().keys()) | set(__all__))
