"""MI355X-native partition-overlap layer engine."""

from .block import DecoderLayer, LayerConfig, LayerStack
from .block_scaled import BlockOperand, BlockScaled
from .model import GPTModelShard, LanguageModelEmbedding

__all__ = ["BlockOperand", "BlockScaled", "DecoderLayer", "GPTModelShard", "LanguageModelEmbedding", "LayerConfig", "LayerStack"]
__version__ = "0.1.0"
