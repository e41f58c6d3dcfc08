"""MI355X-native partition-overlap layer engine."""

from .block import DecoderLayer, LayerConfig, LayerStack
from .block_scaled import BlockOperand, BlockScaled
from .gradients import clip_grad_norm, grad_norm
from .model import GPTModelShard, LanguageModelEmbedding
from .rotary_axes import RotaryAxes, rotary_axes

__all__ = ["BlockOperand", "BlockScaled", "DecoderLayer", "GPTModelShard", "LanguageModelEmbedding", "LayerConfig", "LayerStack",
           "RotaryAxes", "clip_grad_norm", "grad_norm", "rotary_axes"]
__version__ = "0.1.0"
