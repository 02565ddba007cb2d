"""quant_cast_cuda: the CUDA backend of the quant-cast recipes (a sibling of quant_cast_triton /
quant_cast_cute in vkuzo/quant_cast_bench)."""
from .recipes import *  # noqa: F401,F403
from .recipes import ALL_RECIPES, QuantCastCudaRecipe  # noqa: F401
from .int8_linear import int8_scaled_mm_cuda, rowwise_int8_cuda  # noqa: F401
from .kv_cache import (nvfp4_kv_append_cuda, nvfp4_kv_attention_cuda, nvfp4_kv_cache_cuda,  # noqa: F401
                       nvfp4_kv_gather_cuda)
from ._lib import get_scalar_division, scalar_division, set_scalar_division  # noqa: F401
