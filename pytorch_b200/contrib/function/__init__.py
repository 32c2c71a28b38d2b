from .quantized_mlp import w8a8_swiglu_mlp  # noqa: F401
from .quantized_moe import w8a8_swiglu_moe  # noqa: F401
