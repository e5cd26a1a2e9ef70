from .attention import structure_attention
from .dropout import CounterDropout, counter_dropout
from .embedding import ScaledEmbedding, embedding_lookup

__all__ = ["structure_attention", "counter_dropout", "CounterDropout", "embedding_lookup", "ScaledEmbedding"]
