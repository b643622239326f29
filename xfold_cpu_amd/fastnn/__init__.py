"""HIP operators behind the reference's fastnn API (``xfold/fastnn/__init__.py:1-5``), and the ones with
a backward pass beside them: ``trainable_layer_norm`` and ``sequence_attention``."""

from .layer_norm import LayerNorm, trainable_layer_norm
from .attention import dot_product_attention
from .gated_linear_unit import gated_linear_unit
from .sequence import sequence_attention

__all__ = ["LayerNorm", "dot_product_attention", "gated_linear_unit", "sequence_attention", "trainable_layer_norm"]
