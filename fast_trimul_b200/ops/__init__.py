from .triangle import FastTriangleMultiplication  # noqa: F401
from .norm import FastLayerNorm, layer_norm  # noqa: F401
