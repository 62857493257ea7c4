from .conditional_transformer import RPEConditionalTransformer
from .differential_transformer import (DifferentialAttentionLayer, DifferentialConditionalTransformer, DifferentialMultiHeadAttention,
                                       DifferentialTransformerLayer, differential_attention)
from .output_layer import AttentionOutput
from .positional_embedding import SinusoidalPositionalEmbedding
from .rotary_embedding import RotaryPositionalEmbedding, rotary_frequencies
from .rpe_transformer import RPEAttentionLayer, RPEMultiHeadAttention, RPETransformerLayer
from .vanilla_transformer import AttentionLayer, MultiHeadAttention, TransformerLayer
