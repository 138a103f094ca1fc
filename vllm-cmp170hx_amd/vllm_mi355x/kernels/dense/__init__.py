"""Linear layers of plain 16-bit weights on gfx950: routers, shared experts and the
layers that a quantized model leaves as they are.  No counterpart in the reference."""

from .ops import dense_linear

__all__ = ["dense_linear"]
