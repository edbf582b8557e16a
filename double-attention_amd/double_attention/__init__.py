"""MI355X-native shared-dictionary attention (drop-in for ``double_attention``).

Public names follow the reference package's API (reference
``src/double_attention/__init__.py:1-47``) for the attention path; the
additions are ``backend="hip"`` in the config, ``HIP_AVAILABLE``, the gfx950
operator functions ``dictionary_route_hip`` / ``routed_attention_hip``, and
the 8-bit operators of the feed-forward (``int8_ops``).
"""

from . import _lib
from .checkpoint import GraphedForward, load_model_from_checkpoint, load_training_checkpoint
from .config import DoubleAttentionConfig, experiment_config, experiment_names
from .hip_ops import dictionary_normalize_hip, dictionary_route_hip, routed_attention_hip
from .int8_ops import (
    INT8_GROUP,
    QuantizedRows,
    add_rms_norm_backward_hip,
    add_rms_norm_hip,
    add_rms_norm_int8_hip,
    dequantize_int8_hip,
    gelu_int8_backward_hip,
    gelu_int8_hip,
    linear_int8_hip,
    quantize_int8_hip,
)
from .modules import (
    DoubleAttentionAux,
    DoubleAttentionBlock,
    DoubleAttentionLM,
    DoubleAttentionStack,
    SharedDictionaryAttention,
    SharedDictionaryBank,
)
from .ops import assemble_score_maps, dictionary_route_reference, routed_attention_reference
from .triton_kernels import TRITON_AVAILABLE

HIP_AVAILABLE = _lib.available()

__all__ = [
    "DoubleAttentionAux",
    "DoubleAttentionBlock",
    "DoubleAttentionConfig",
    "DoubleAttentionLM",
    "DoubleAttentionStack",
    "GraphedForward",
    "HIP_AVAILABLE",
    "INT8_GROUP",
    "QuantizedRows",
    "SharedDictionaryAttention",
    "SharedDictionaryBank",
    "TRITON_AVAILABLE",
    "add_rms_norm_backward_hip",
    "add_rms_norm_hip",
    "add_rms_norm_int8_hip",
    "assemble_score_maps",
    "dequantize_int8_hip",
    "dictionary_normalize_hip",
    "dictionary_route_hip",
    "dictionary_route_reference",
    "experiment_config",
    "experiment_names",
    "gelu_int8_backward_hip",
    "gelu_int8_hip",
    "linear_int8_hip",
    "load_model_from_checkpoint",
    "load_training_checkpoint",
    "quantize_int8_hip",
    "routed_attention_hip",
    "routed_attention_reference",
]
