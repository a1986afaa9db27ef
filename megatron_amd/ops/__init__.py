"""HIP/CDNA4 ops for MI355X (gfx950).

functional: autograd ops (rmsnorm, layernorm, softmax, glu, rope,
bias_dropout_add, flash attention, rotary, sampling) dispatching to the in-tree
_C.so. quant_kv: key/value cache in 4 bits and the attention over it.
ext: extension loader. build: ahead-of-time hipcc build driver.
"""

from . import ext  # noqa: F401
from .functional import (  # noqa: F401
    apply_rope,
    bias_dropout_add,
    flash_attention,
    glu_activation,
    layernorm,
    rmsnorm,
    rotary_embedding,
    sample_tokens,
    scaled_masked_softmax,
    swiglu,
)
from .quant_kv import QuantKVCache  # noqa: F401
